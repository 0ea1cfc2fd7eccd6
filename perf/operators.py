"""The readout at training scale and in 8 bits: what its operators are measured on.

  score       noetic_rl.readout_score_with_stats: each position's token log-probability (minus the
              cross entropy over the vocabulary), its log-sum-exp and, where asked for, its entropy,
              from the hidden states and the readout's weight, the logits never kept.
  train       the same followed by noetic_rl.readout_score_grad: the gradients of
              sum g_logp logp + g_entropy entropy with respect to the hidden states and the weight.
  checkpoint  noetic_ops.quantize_int8 and noetic_ops.dequantize_int8: rows (or, through a swapped view,
              columns) held as 8-bit integers with a scale each, and what they stand for.
  linear8     noetic_ops.quantize_int8 of the activations, a scale for each token, and
              noetic_ops.matmul_int8 with a weight quantized once, a scale for each channel.

With x = hidden . W, z = x / tau (+ mask; a token whose u8 mask is 0 is excluded), base = max z,
rest = ln sum exp(z - base): logp = z[token] - base - rest, entropy = -sum p ln p, p = exp(z - base - rest),
d/dz = g_logp (onehot - p) - g_entropy p (ln p + entropy), d/dx = d/dz / tau, d_hidden = d/dx . W^T,
d_weight = hidden^T . d/dx. A quantized row is q = round(x / s), ties to even, s = max |x| / 127 in f32.

A weight is "dv" [dim, vocab] or "vd" [vocab, dim].
"""
import math
import os
import sys

import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # scoring one step's tokens of a small decode batch: the latency of the smallest training readout
        {"name": "score_step", "op": "score", "rows": 64, "dim": 1024, "vocab": 32000, "dtype": "bf16", "layout": "dv",
         "mask": "none", "tau": 0.8, "entropy": False},
        # scoring a rollout of 4096 positions at the benchmark's large vocabulary and head width
        {"name": "score_rollout", "op": "score", "rows": 4096, "dim": 4096, "vocab": 128256, "dtype": "bf16",
         "layout": "vd", "mask": "none", "tau": 1.0, "entropy": True},
        # a ragged f16 batch of positions under a random keep-mask
        {"name": "score_masked", "op": "score", "rows": 1000, "dim": 1000, "vocab": 50257, "dtype": "f16",
         "layout": "dv", "mask": "u8", "tau": 0.7, "entropy": True},
        # one micro-batch of a small model's language-model loss with its gradients
        {"name": "train_small", "op": "train", "rows": 128, "dim": 1024, "vocab": 32000, "dtype": "bf16", "layout": "vd",
         "mask": "none", "tau": 1.0, "entropy": False},
        # a policy update with an entropy bonus under one additive vocabulary mask
        {"name": "train_policy", "op": "train", "rows": 2048, "dim": 4096, "vocab": 50304, "dtype": "bf16",
         "layout": "dv", "mask": "f32_shared", "tau": 0.8, "entropy": True},
        # the loss and its gradients of a large training step
        {"name": "train_large", "op": "train", "rows": 4096, "dim": 4096, "vocab": 128256, "dtype": "bf16",
         "layout": "vd", "mask": "none", "tau": 1.0, "entropy": False},
        # odd sizes throughout, f16, a keep-mask row for each position
        {"name": "train_odd", "op": "train", "rows": 333, "dim": 1001, "vocab": 50257, "dtype": "f16", "layout": "dv",
         "mask": "u8", "tau": 0.7, "entropy": True},
        # a layer's activations kept in 8 bits between the forward and the backward pass
        {"name": "checkpoint_tokens", "op": "checkpoint", "rows": 4096, "cols": 4096, "dtype": "bf16",
         "by": "rows"},
        # a [dim, vocab] readout weight of f32, a scale for each output channel
        {"name": "checkpoint_channels", "op": "checkpoint", "rows": 1024, "cols": 50304, "dtype": "f32",
         "by": "columns"},
        # the readout of a single decoded token
        {"name": "linear8_token", "op": "linear8", "m": 1, "k": 4096, "n": 128256, "dtype": "bf16", "out": "f32"},
        # the readout of a decode batch
        {"name": "linear8_batch", "op": "linear8", "m": 64, "k": 4096, "n": 50304, "dtype": "bf16", "out": "bf16"},
        # a projection over a whole prompt
        {"name": "linear8_prompt", "op": "linear8", "m": 4096, "k": 4096, "n": 16384, "dtype": "bf16", "out": "bf16"},
    ]


def _size(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _even_out(rng, v):
    """v itself, or v as a multiple of 8 or 64."""
    pad = rng.choice([1, 8, 64])
    return max(v // pad, 1) * pad


def draw(rng):
    op = rng.choice(["score", "score", "train", "train", "train", "checkpoint", "linear8", "linear8"])
    if op in ("score", "train"):
        vocab = rng.choice([32000, 50304, 128256, 151936]) if rng.random() < 0.3 else _even_out(rng, _size(rng, 1000, 152000))
        dim = rng.choice([1024, 2048, 4096]) if rng.random() < 0.3 else _even_out(rng, _size(rng, 64, 4096))
        rows = _size(rng, 1, min(8192, 4096 * 4096 * 128256 // (dim * vocab)))
        return {"op": op, "rows": rows, "dim": dim, "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "f16"]),
                "layout": rng.choice(["dv", "vd"]), "mask": rng.choice(["none", "none", "u8", "f32_shared"]),
                "tau": rng.choice([0.6, 0.7, 0.8, 1.0]), "entropy": rng.random() < 0.5}
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "checkpoint":
        cols = _size(rng, 1, 16384)
        rows = _size(rng, 1, min(65536, 100_000_000 // cols))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "by": rng.choice(["rows", "rows", "columns"])}
    k, n = _even_out(rng, _size(rng, 16, 16384)), _even_out(rng, _size(rng, 100, 128256))
    m = _size(rng, 1, min(8192, 4096 * 4096 * 16384 // (k * n)))
    return {"op": op, "m": m, "k": k, "n": n, "dtype": dtype, "out": rng.choice(["f32", "bf16", "f16"])}


# ------------------------------------------------------------------------------------- inputs

def _normal(shape, dtype, g, std):
    return torch.empty(shape, dtype=_TORCH[dtype], device="cuda").normal_(0.0, std, generator=g)


def _inputs(case, seed):
    """Every input as torch tensors, a function of the case and the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] in ("score", "train"):
        R, d, V = case["rows"], case["dim"], case["vocab"]
        x = {"hidden": _normal((R, d), case["dtype"], g, 1.0),
             "weight": _normal((d, V) if case["layout"] == "dv" else (V, d), case["dtype"], g, 2.0 / math.sqrt(d)),
             "tokens": torch.randint(0, V, (R,), device="cuda", generator=g, dtype=torch.int32), "mask": None}
        if case["mask"] != "none":
            n = R if case["mask"] == "u8" else 1
            keep = torch.rand((n, V), device="cuda", generator=g) < 0.9
            keep[torch.arange(R, device="cuda") if n > 1 else 0, x["tokens"].long()] = True  # scored tokens are allowed
            x["mask"] = keep.to(torch.uint8) if case["mask"] == "u8" else torch.where(keep, 0.0, -math.inf)
        if case["op"] == "train":  # a policy gradient's weights over the positions, f16 ones under a loss scale
            share = (1024.0 if case["dtype"] == "f16" else 1.0) / R
            x["g_logp"] = torch.randn(R, device="cuda", generator=g) * share
            x["g_entropy"] = torch.full((R,), 0.01 * share, device="cuda") if case["entropy"] else None
        return x
    if case["op"] == "checkpoint":
        x = _normal((case["rows"], case["cols"]), case["dtype"], g, 1.0)
        return {"x": x.mul_(torch.rand((case["rows"], 1), device="cuda", generator=g).mul_(4.0).exp_())}
    x = {"x": _normal((case["m"], case["k"]), case["dtype"], g, 1.0)}
    w = _normal((case["n"], case["k"]), "f32", g, 1.0 / math.sqrt(case["k"]))
    x["w_scale"] = (w.abs().amax(1).double() / 127.0).float()
    x["w"] = torch.round(w / x["w_scale"][:, None]).clamp_(-127, 127).to(torch.int8)
    return x


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# ------------------------------------------------------------------------------------- the plain forms

def _logits(s):
    case = s["case"]
    w = s["weight"].float()
    z = s["hidden"].float() @ (w if case["layout"] == "dv" else w.t())
    z /= case["tau"]
    if case["mask"] == "u8":
        z.masked_fill_(s["mask"] == 0, -math.inf)
    elif case["mask"] != "none":
        z += s["mask"]
    return z, w


def _score(s):
    z, w = _logits(s)
    at = s["tokens"].long()[:, None]
    base = z.amax(1)
    z -= base[:, None]
    rest = z.exp().sum(1).log()
    z -= rest[:, None]  # ln p
    out = {"logp": z.gather(1, at)[:, 0], "base": base, "rest": rest}
    if s["case"]["entropy"]:
        out["entropy"] = -torch.where(z == -math.inf, 0.0, z.exp() * z).sum(1)
    return out, z, w


def _train(s):
    out, lnp, w = _score(s)
    case = s["case"]
    p = lnp.exp()
    dz = p * -s["g_logp"][:, None]
    if case["entropy"]:
        dz -= torch.where(p == 0, 0.0, p * (lnp + out["entropy"][:, None])) * s["g_entropy"][:, None]
    dz.scatter_add_(1, s["tokens"].long()[:, None], s["g_logp"][:, None])
    dz /= case["tau"]
    h = s["hidden"].float()
    if case["layout"] == "dv":
        d_hidden, d_weight = dz @ w.t(), h.t() @ dz
    else:
        d_hidden, d_weight = dz @ w, dz.t() @ h
    return dict(out, d_hidden=d_hidden.to(s["hidden"].dtype), d_weight=d_weight.to(s["weight"].dtype))


def _quantized(x):
    """q (as whole f32 values) and the scale of each row; the quotient in 64 bits, for a value next to a border."""
    scale = (x.abs().amax(1).double() / 127.0).float()
    return torch.round(x.double() / scale.double()[:, None]).float(), scale


def _checkpoint(s):
    x = s["x"].t() if s["case"]["by"] == "columns" else s["x"]
    q, scale = _quantized(x)
    return {"values": (q * scale[:, None]).to(x.dtype), "scale": scale}


def _linear8(s):
    q, scale = _quantized(s["x"])
    y = (q @ s["w"].float().t()) * scale[:, None] * s["w_scale"]
    return y.to(_TORCH[s["case"]["out"]])


# ------------------------------------------------------------------------------------- the framework's operators

class _Held:
    """A torch allocation as the buffer behind a noetic_rl.Tensor."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


class _Export:
    def __init__(self, t):
        self.owner = t
        kind = {"f32": "<f4", "bf16": "<i2", "f16": "<f2"}[t.dtype]
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": kind, "data": (t.ptr, False), "version": 2}


_NAMES = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16", torch.int8: "i8", torch.uint8: "u8",
          torch.int32: "i32"}


def _framework():
    at = os.path.join(os.getcwd(), "noetic-tensor_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import noetic_ops
    import noetic_rl
    return noetic_rl, noetic_ops


def _given(nr, t):
    """A contiguous torch tensor as the library's device tensor, in place."""
    return None if t is None else nr.Tensor(tuple(t.shape), _NAMES[t.dtype], _Held(t))


def _taken(t):
    """The library's device tensor as a torch tensor over the same memory (kept alive by it)."""
    x = torch.as_tensor(_Export(t), device="cuda")
    return x.view(torch.bfloat16) if t.dtype == "bf16" else x


def _own_readout(s):
    nr, _ = _framework()
    case = s["case"]
    hidden, weight, mask, tokens = (_given(nr, s[k]) for k in ("hidden", "weight", "mask", "tokens"))
    with nr.matmul_precision_scope(nr.MatmulPrecision.HALF):
        logp, entropy, stats = nr.readout_score_with_stats(hidden, weight, case["tau"], mask, tokens,
                                                           entropy=case["entropy"], layout=case["layout"], check=False)
        out = {"logp": logp, "base": stats.lse_base, "rest": stats.lse_rest}
        if case["entropy"]:
            out["entropy"] = entropy
        if case["op"] == "train":
            out["d_hidden"], out["d_weight"] = nr.readout_score_grad(
                hidden, weight, case["tau"], mask, tokens, stats, entropy=entropy, g_logp=_given(nr, s["g_logp"]),
                g_entropy=_given(nr, s["g_entropy"]), layout=case["layout"])
    return {k: _taken(v) for k, v in out.items()}


def _own_checkpoint(s):
    nr, ops = _framework()
    x = _given(nr, s["x"])
    view = ops.Layout.contiguous(x.shape)
    q, scale = ops.quantize_int8(x, view.swapped(0, 1) if s["case"]["by"] == "columns" else view)
    return {"values": _taken(ops.dequantize_int8(q, scale, s["case"]["dtype"])), "scale": _taken(scale)}


def _own_linear8(s):
    nr, ops = _framework()
    x = _given(nr, s["x"])
    q, scale = ops.quantize_int8(x, ops.Layout.contiguous(x.shape))
    return _taken(ops.matmul_int8(q, scale, _given(nr, s["w"]), _given(nr, s["w_scale"]), s["case"]["out"]))


def run(s):
    op = s["case"]["op"]
    if own:
        return {"score": _own_readout, "train": _own_readout, "checkpoint": _own_checkpoint,
                "linear8": _own_linear8}[op](s)
    if op == "score":
        return _score(s)[0]
    return {"train": _train, "checkpoint": _checkpoint, "linear8": _linear8}[op](s)


# ------------------------------------------------------------------------------------- work and 64 bits

def work(case):
    """Each input read once and each output written once; the products once each (the logits, and for the
    gradients one with the weight and one with the hidden states)."""
    if case["op"] in ("score", "train"):
        R, d, V = case["rows"], case["dim"], case["vocab"]
        b = 2 * R * d + 2 * V * d + {"none": 0, "u8": R * V, "f32_shared": 4 * V}[case["mask"]] + 20 * R
        if case["op"] == "score":
            return {"bytes": b, "flops": 2 * R * V * d}
        return {"bytes": b + 2 * R * d + 2 * V * d + 4 * R, "flops": 6 * R * V * d}
    if case["op"] == "checkpoint":  # the values in, their 8 bits out and in, the values out
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * _SIZE[case["dtype"]] + 2) + 8 * (case["rows"] if case["by"] == "rows" else case["cols"]),
                "flops": 0}
    m, k, n = case["m"], case["k"], case["n"]
    return {"bytes": m * k * _SIZE[case["dtype"]] + n * k + 4 * n + m * n * _SIZE[case["out"]], "flops": 2 * m * k * n}


def _readout64(case, x):
    W = x["weight"].double()
    if case["layout"] == "vd":
        W = W.t().contiguous()
    h = x["hidden"].double()
    z = torch.matmul(h, W).div_(case["tau"])
    if x["mask"] is not None:
        z[(x["mask"] == (0 if case["mask"] == "u8" else -math.inf)).expand_as(z)] = -math.inf
    lse = torch.logsumexp(z, 1, keepdim=True)
    base = z.max(1)[0]
    rows = torch.arange(case["rows"], device="cuda")
    at = x["tokens"].long()
    lnp = z.sub_(lse)
    out = {"logp": lnp[rows, at], "base": base, "rest": lse[:, 0] - base}
    p = lnp.exp()
    plnp = torch.xlogy(p, p)
    if case["entropy"]:
        out["entropy"] = -plnp.sum(1)
    if case["op"] == "score":
        return out
    gl = x["g_logp"].double()
    if case["entropy"]:
        ge = x["g_entropy"].double()
        p = p.mul_((gl + ge * out["entropy"])[:, None]).add_(plnp.mul_(ge[:, None])).neg_()
    else:
        p = p.mul_(-gl[:, None])
    p[rows, at] += gl
    p.div_(case["tau"])
    d_weight = torch.matmul(h.t().contiguous(), p)
    return dict(out, d_hidden=torch.matmul(p, W.t().contiguous()),
                d_weight=d_weight if case["layout"] == "dv" else d_weight.t().contiguous())


def exact(case, seed):
    """run()'s outputs in 64 bits from torch alone; the scales are what they are in f32."""
    x = _inputs(case, seed)
    if case["op"] in ("score", "train"):
        return _readout64(case, x)
    v = x["x"].double()
    if case.get("by") == "columns":
        v = v.t().contiguous()
    s = torch.div(v.abs().max(1, keepdim=True)[0], 127.0).float().double()
    q = torch.div(v, s).round_()
    if case["op"] == "checkpoint":
        return {"values": q * s, "scale": s[:, 0]}
    return torch.matmul(q, x["w"].double().t().contiguous()) * s * x["w_scale"].double()
