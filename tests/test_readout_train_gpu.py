"""The training readout (nt_hip_rl_readout_score_stats, nt_hip_rl_readout_score_backward) against the same
formulas in 64 bits on the operands' own values.

Tolerances, from the arithmetic. A logit is an f32 sum of d products of 16-bit values, exact each: off by at most
dz = (d + 8) 2^-24 sum |h||w| / tau (8 more roundings: the temperature, the mask, y's own). A log-probability or a
log-sum-exp is off by 2 dz and its own f32 roundings; the sum of exponentials' terms by the hardware's exp2, 2^-22 of
each. A probability is off by 2 dz + 2^-21 of itself. G is rounded once, by u = eps/2 of the type, and so is a
gradient; a gradient's f32 sum of n terms is off by n 2^-24 of the sum of their magnitudes. An f16 gradient has
steps of 2^-24 at the least, and its G steps of 2^-24 of the row's unit; a bf16 G, a probability and a bf16 gradient
under 2^-126, the smallest normal value, count as zero: the matrix cores and the hardware's exp2 take no smaller ones."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import noetic_ops as ops
import noetic_rl as nr
from tests.test_kept_blocks_gpu import Capture

pytestmark = pytest.mark.gpu

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {t: torch.finfo(TORCH[t]).eps / 2 for t in TORCH}


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    prev = nr.set_matmul_precision(nr.MatmulPrecision.HALF)
    yield
    nr.set_matmul_precision(prev)


def given(a, dtype=None):
    """A CPU torch or numpy value as a device tensor."""
    if isinstance(a, torch.Tensor):
        name = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32", torch.int32: "i32",
                torch.uint8: "u8"}[a.dtype]
        b = a.contiguous().view(torch.int16).numpy().view(np.uint16) if name in TORCH else a.contiguous().numpy()
        return nr.Tensor.from_numpy(b, name)
    return nr.Tensor.from_numpy(a, dtype)


def values(t):
    return torch.from_numpy(t.to_f64())


class Case:
    """Inputs on the host; the mask as given and as what is added to z."""

    def __init__(self, rows, V, d, dtype="bf16", layout="dv", mask="none", tau=1.0, entropy=True, seed=0, scale=2.0):
        g = torch.Generator().manual_seed(1000 * rows + 10 * V + d + seed)
        self.rows, self.V, self.d, self.dtype, self.layout, self.tau, self.entropy = rows, V, d, dtype, layout, tau, entropy
        self.h = torch.randn(rows, d, generator=g).to(TORCH[dtype])
        w = (torch.randn(V, d, generator=g) * scale / math.sqrt(d)).to(TORCH[dtype])
        self.w = w if layout == "vd" else w.t().contiguous()
        self.tokens = torch.randint(0, V, (rows,), generator=g, dtype=torch.int32)
        self.g_logp = torch.randn(rows, generator=g) / max(rows, 1) * (256.0 if dtype == "f16" else 1.0)
        self.g_entropy = torch.randn(rows, generator=g) * 0.1 / max(rows, 1) * (256.0 if dtype == "f16" else 1.0)
        self.mask, self.add = None, torch.zeros(1, V, dtype=torch.float64)
        if mask != "none":
            n = 1 if mask.endswith("shared") else rows
            keep = torch.rand(n, V, generator=g) < 0.6
            keep[torch.arange(rows) if n == rows else 0, self.tokens.long()] = True
            if mask.startswith("u8"):
                self.mask = keep.to(torch.uint8) * 3  # (any value but 0 keeps)
                self.add = torch.where(keep, 0.0, -math.inf).double()
            else:
                low = -1e9 if "low" in mask else (torch.finfo(torch.float32).min if "least" in mask else -math.inf)
                m = torch.where(keep, torch.randn(n, V, generator=g) if "bias" in mask else torch.zeros(n, V), low)
                self.mask = m.bfloat16() if "bf16" in mask else m
                self.add = self.mask.double()

    def run(self, check=True):
        h, w, m, t = given(self.h), given(self.w), None if self.mask is None else given(self.mask), given(self.tokens)
        lp, ent, stats = nr.readout_score_with_stats(h, w, self.tau, m, t, entropy=self.entropy, layout=self.layout,
                                                     check=check)
        gh, gw = nr.readout_score_grad(h, w, self.tau, m, t, stats, entropy=ent, g_logp=given(self.g_logp),
                                       g_entropy=given(self.g_entropy) if self.entropy else None, layout=self.layout)
        out = {"logp": lp, "base": stats.lse_base, "rest": stats.lse_rest, "grad_hidden": gh, "grad_weight": gw}
        if self.entropy:
            out["entropy"] = ent
        return out

    def want(self):
        """The formulas in 64 bits, and how far each value may be off."""
        h, w = self.h.double(), self.w.double()
        w = w.t() if self.layout == "vd" else w  # [d, V]
        z = h @ w / self.tau + self.add
        dz = (self.d + 8) * 2.0 ** -24 * (h.abs() @ w.abs() / self.tau + torch.where(self.add.isfinite(), self.add.abs(), 0.0))
        dz = dz.amax(1, keepdim=True) if self.V else dz
        rows, at = torch.arange(self.rows), self.tokens.long()
        lse = torch.logsumexp(z, 1, keepdim=True)
        lnp = z - lse
        p = lnp.exp()
        plnp = torch.xlogy(p, p)
        H = -plnp.sum(1, keepdim=True)
        gl = self.g_logp.double()[:, None]
        ge = self.g_entropy.double()[:, None] * (1.0 if self.entropy else 0.0)
        one = torch.zeros_like(p)
        one[rows, at] = 1.0
        G = (gl * (one - p) - ge * (plnp + p * H)) / self.tau
        f32 = 2.0 ** -22
        out = {"logp": lnp[rows, at], "base": z.amax(1), "rest": (lse - z.amax(1, keepdim=True))[:, 0], "entropy": H[:, 0]}
        tol = {"logp": 2 * dz[:, 0] + f32 * (out["logp"].abs() + lse[:, 0].abs() + 1),
               "base": dz[:, 0] + f32 * (out["base"].abs() + 1), "rest": 2 * dz[:, 0] + f32 * (lse[:, 0].abs() + 2)}
        # an entropy: each term's p off by dp, times |ln p| and with ln p off by 2 dz
        dp = 2 * dz + 2.0 ** -21
        tol["entropy"] = (dp * plnp.abs()).sum(1) + 2 * dz[:, 0] + f32 * (1 + H[:, 0])
        # G: rounded once; p off by dp, ln p by 2 dz; f16: steps of 2^-24 of a unit of 2^(e - 14)
        u = HALF_STEP[self.dtype]
        size = gl.abs() * p + ge.abs() * (plnp.abs() + p * (H + 1))
        dG = (u + 2.0 ** -22) * G.abs() + (2 * dp + 2 * tol["entropy"][:, None] + 2.0 ** -21) * size / self.tau
        unit = torch.zeros_like(gl)
        if self.dtype == "f16":
            unit = 2.0 ** torch.ceil(torch.log2((gl.abs() + 16 * ge.abs()).clamp(min=1e-30)) + 1e-9) * 2.0
            dG = dG + 2.0 ** -38 * unit / self.tau
        else:
            dG = dG + 2.0 ** -126 * (1 + (gl.abs() + ge.abs() * (H + 88)) / self.tau)  # (G's own, and p's times its factor)
        aw, ah = w.abs(), h.abs()
        out["grad_hidden"] = G @ w.t()
        sums = G.abs() @ aw.t()
        tol["grad_hidden"] = dG @ aw.t() + self.V * 2.0 ** -24 * sums + u * out["grad_hidden"].abs()
        gw = h.t() @ G
        tw = ah.t() @ dG + self.rows * 2.0 ** -24 * (ah.t() @ G.abs()) + u * gw.abs()
        if self.dtype == "f16":
            tol["grad_hidden"] = tol["grad_hidden"] + 2.0 ** -25
            # a row of H scaled by 2^(e - top) has steps of 2^-24 itself
            tw = tw + 2.0 ** -25 + 2.0 ** -25 * float(unit.max()) * (G.abs() / unit.clamp(min=1e-30)).sum(0)[None, :]
        else:
            tol["grad_hidden"], tw = tol["grad_hidden"] + 2.0 ** -126, tw + 2.0 ** -126
        out["grad_weight"], tol["grad_weight"] = (gw, tw) if self.layout == "dv" else (gw.t(), tw.t())
        return out, tol


def agree(got, want, tol, name):
    got, want = got.reshape(want.shape), want.double()
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: NaNs"
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]), f"{name}: infinities"
    off = (got - want).abs()[fine] - tol.expand_as(want)[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{name}: {off.max():.3g} past the tolerance, at {int((off > 0).sum())} places"


def check(case):
    got, (want, tol) = case.run(), case.want()
    for k in got:
        agree(values(got[k]), want[k], tol[k], k)
    return got


SIZES = [(1, 1, 1), (1, 2, 8), (2, 3, 5), (3, 257, 16), (64, 1000, 64), (65, 511, 72), (129, 1031, 33), (300, 2050, 264),
         (256, 256, 64), (257, 640, 96), (17, 5003, 1001)]


@pytest.mark.parametrize("layout", ["dv", "vd"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,V,d", SIZES)
def test_sizes(rows, V, d, dtype, layout):
    check(Case(rows, V, d, dtype, layout, tau=0.8))


@pytest.mark.parametrize("mask", ["u8", "u8_shared", "f32", "f32_shared", "f32_bias", "f32_low", "f32_least", "bf16_bias"])
@pytest.mark.parametrize("rows,V,d,dtype,layout", [(70, 1003, 40, "bf16", "dv"), (5, 640, 64, "f16", "vd")])
def test_masks(rows, V, d, dtype, layout, mask):
    check(Case(rows, V, d, dtype, layout, mask, tau=0.7))


@pytest.mark.parametrize("tau", [0.05, 1.0, 3.7])
def test_without_entropy_and_temperatures(tau):
    check(Case(40, 900, 48, tau=tau, entropy=False))


def test_large_logits():
    """Logits in the hundreds: one token takes nearly all of each row."""
    check(Case(50, 700, 64, scale=60.0))


def test_pieces_of_the_vocabulary():
    """G of 4100 rows and 70000 columns is past 512 MiB: two pieces, the second shorter; a sample of the gradients."""
    c = Case(4100, 70000, 16, "bf16", "vd", entropy=False)
    got = c.run()
    dev = "cuda"
    h, w = c.h.double().to(dev), c.w.double().to(dev)
    z = h @ w.t()
    lse = torch.logsumexp(z, 1, keepdim=True)
    at = c.tokens.long().to(dev)
    G = (z - lse).exp_().mul_(-c.g_logp.double().to(dev)[:, None])
    G[torch.arange(c.rows, device=dev), at] += c.g_logp.double().to(dev)
    u = HALF_STEP["bf16"]
    for name, want, size in (("grad_hidden", G @ w, G.abs() @ w.abs()), ("grad_weight", G.t() @ h, G.abs().t() @ h.abs())):
        off = (values(got[name]).to(dev) - want).abs() - (u + 2.0 ** -12 + c.V * 2.0 ** -24) * size - u * want.abs()  # (dp under 2^-12 here)
        assert off.max() <= 0, name


def test_gradients_against_differences():
    """d(sum g_logp logp + g_entropy entropy) along a direction, from the forward's own values a step apart on each
    side, in f16 operands whose steps are exact (a difference of second order: step^2, and the forward's f32)."""
    c = Case(12, 300, 32, "f16", "vd", tau=0.9)
    got = {k: values(v) for k, v in c.run().items()}
    g = torch.Generator().manual_seed(5)

    def loss(h, w):
        c2 = Case(12, 300, 32, "f16", "vd", tau=0.9)
        c2.h, c2.w = h, w
        o = c2.want()[0]
        return float((c.g_logp.double() * o["logp"] + c.g_entropy.double() * o["entropy"]).sum())

    for name, x, at in (("grad_hidden", c.h, 0), ("grad_weight", c.w, 1)):
        step = torch.randint(-1, 2, x.shape, generator=g).to(torch.float16) * 2.0 ** -7
        up, down = x + step, x - step
        move = up.double() - down.double()
        pair = lambda v: (v, c.w) if at == 0 else (c.h, v)  # noqa: E731
        diff = loss(*pair(up)) - loss(*pair(down))
        along = float((got[name].reshape(x.shape) * move).sum())
        size = float((got[name].reshape(x.shape).abs() * move.abs()).sum())
        assert abs(diff - along) <= 2.0 ** -9 * size, (name, diff, along, size)


# ----------------------------------------------------------------------------- rows that are not plain

def test_rows_without_a_token_bad_tokens_and_padding():
    c = Case(40, 500, 24, "bf16", "dv", "u8", tau=0.8)
    c.mask[7] = 0                      # nothing allowed
    c.mask[9, int(c.tokens[9])] = 0    # the scored token excluded
    c.tokens[11], c.tokens[13] = -1, 500
    c.h[20] = math.nan                 # a padded position: nothing flows through it
    c.h[21, 3] = math.inf
    c.g_logp[20:22] = 0.0
    c.g_entropy[20:22] = 0.0
    h, w, m, t = given(c.h), given(c.w), given(c.mask), given(c.tokens)
    with pytest.raises(IndexError, match="out of range 500 at position 11"):
        nr.readout_score_with_stats(h, w, c.tau, m, t)
    got = {k: values(v) for k, v in c.run(check=False).items()}
    # the same rows without what is wrong with them
    d = Case(40, 500, 24, "bf16", "dv", "u8", tau=0.8)
    d.mask, d.add = c.mask.clone(), torch.where(c.mask > 0, 0.0, -math.inf).double()
    d.mask[7], d.add[7] = 1, 0.0
    d.h[20:22] = 0.0
    d.g_logp[[7, 11, 13, 20, 21]] = 0.0
    d.g_entropy[[7, 20, 21]] = 0.0
    want, tol = d.want()
    for k in ("logp", "entropy", "base", "rest"):
        w_, t_ = want[k].clone(), tol[k].clone()
        w_[[7, 20, 21]] = math.nan
        if k == "logp":
            w_[[11, 13]] = math.nan
            assert w_[9] == -math.inf
        if k in ("base", "rest"):
            w_[7] = -math.inf if k == "base" else 0.0
        agree(got[k], w_, t_.nan_to_num(0.0), k)
    # the excluded token's own term flows all the same, as the op sequence's does
    for k in ("grad_hidden", "grad_weight"):
        agree(got[k], want[k], tol[k], k)
    assert (got["grad_hidden"][[7, 20, 21]] == 0).all()


def test_a_nan_row_with_a_gradient_is_nan():
    c = Case(8, 100, 16)
    c.h[3, 5] = math.nan
    got = {k: values(v) for k, v in c.run().items()}
    assert got["logp"].isnan().tolist() == [i == 3 for i in range(8)]
    assert got["grad_hidden"].isnan().any(1).tolist() == [i == 3 for i in range(8)]
    assert got["grad_weight"].isnan().all()


def test_no_rows():
    c = Case(0, 100, 16)
    got = c.run()
    assert got["logp"].shape == (0,) and got["grad_hidden"].shape == (0, 16)
    assert (values(got["grad_weight"]) == 0).all()


def test_f16_gradients_of_rows_far_apart():
    """Upstream gradients from 2^-20 to 2^12: each row's hidden gradient keeps its own precision."""
    c = Case(33, 400, 32, "f16", "vd", entropy=False)
    c.g_logp = (2.0 ** torch.linspace(-20, 12, 33)).float()
    got, (want, tol) = c.run(), c.want()
    for k in got:
        agree(values(got[k]), want[k], tol[k], k)


def test_bf16_gradients_of_any_size():
    for s in (1e-30, 1e30):
        c = Case(20, 300, 16, "bf16", "dv")
        c.g_logp, c.g_entropy = c.g_logp * s, c.g_entropy * s
        check(c)


# ----------------------------------------------------------------------------- layout, order, memory

@pytest.mark.parametrize("layout", ["dv", "vd"])
@pytest.mark.parametrize("shift,pad", [(1, 3), (4, 4), (8, 8)])
def test_strides_and_alignment(layout, shift, pad):
    """Operands, masks and gradients inside larger buffers, at every alignment; the padding stays as it was."""
    c = Case(75, 330, 40, "bf16", layout, "f32", tau=0.8)
    wr, wc = c.w.shape

    def inside(x, fill):
        """(device buffer, first element's offset, row stride)."""
        b = torch.full((x.shape[0] * (x.shape[1] + pad) + shift,), fill, dtype=x.dtype)
        rows = b[shift:].view(x.shape[0], x.shape[1] + pad)
        rows[:, :x.shape[1]] = x
        return given(b), shift, x.shape[1] + pad

    (h, oh, ldh), (w, ow, ldw), (m, om, ldm) = inside(c.h, math.nan), inside(c.w, math.nan), inside(c.mask, math.nan)
    t, gl, ge = given(c.tokens), given(c.g_logp), given(c.g_entropy)
    rowf = lambda: nr.Tensor((c.rows,), "f32")  # noqa: E731
    lp, ent, base, rest, st = rowf(), rowf(), rowf(), rowf(), nr.Tensor((c.rows,), "u8")
    lay = nr.NT_READOUT_W_DV if layout == "dv" else nr.NT_READOUT_W_VD
    head = (h.ptr + 2 * oh, w.ptr + 2 * ow, nr.NT_BF16, lay, c.rows, c.V, c.d, ldh, ldw, m.ptr + 4 * om, ldm,
            nr.NT_MASK_F32, 0, c.tau, t.ptr)
    a = nr.NtRlReadoutStatsArgs(*head, lp.ptr, ent.ptr, base.ptr, rest.ptr, st.ptr)
    nr._check(nr.lib().nt_hip_rl_readout_score_stats(C.byref(a)), "stats")
    gh, goh, gldh = inside(torch.full_like(c.h, 7.0), 5.0)
    gw, gow, gldw = inside(torch.full_like(c.w, 7.0), 5.0)
    b = nr.NtRlReadoutStatsGradArgs(*head, base.ptr, rest.ptr, ent.ptr, gl.ptr, ge.ptr, gh.ptr + 2 * goh,
                                    gw.ptr + 2 * gow, gldh, gldw)
    nr._check(nr.lib().nt_hip_rl_readout_score_backward(C.byref(b)), "backward")
    want, tol = c.want()
    for k, v in (("logp", lp), ("entropy", ent), ("base", base), ("rest", rest)):
        agree(values(v), want[k], tol[k], k)
    for k, v, (r, n) in (("grad_hidden", gh, c.h.shape), ("grad_weight", gw, (wr, wc))):
        x = values(v)
        assert (x[:shift] == 5.0).all()
        x = x[shift:].view(r, n + pad)
        assert (x[:, n:] == 5.0).all()
        agree(x[:, :n], want[k], tol[k], k)


@pytest.mark.parametrize("rows", [1, 64, 65, 200, 513])
def test_a_rows_scores_do_not_depend_on_the_others(rows):
    c = Case(rows, 1500, 128, "bf16", "vd", "u8", tau=0.7)
    full = c.run()
    at = [0, rows // 2, rows - 1]
    one = Case(rows, 1500, 128, "bf16", "vd", "u8", tau=0.7)
    one.rows, one.h, one.tokens, one.mask = len(at), c.h[at], c.tokens[at], c.mask[at]
    one.g_logp, one.g_entropy = c.g_logp[at], c.g_entropy[at]
    part = one.run()
    for k in ("logp", "entropy", "base", "rest"):
        assert np.array_equal(full[k].to_numpy()[at], part[k].to_numpy()), k


def test_reruns_are_the_same_bytes():
    c = Case(200, 3000, 200, "f16", "dv", "f32")
    a, b = c.run(), c.run()
    for k in a:
        assert np.array_equal(a[k].to_numpy(), b[k].to_numpy()), k


def test_seeds_and_broadcast_masks():
    """A weight of three seeds: each seed's rows against its own; masks that broadcast over either dimension (the
    rows of a seed as many as the seeds)."""
    S, N, V, d = 3, 3, 260, 32
    parts = [Case(N, V, d, "bf16", "dv", seed=k) for k in range(S)]
    stack = lambda f: torch.stack([getattr(p, f) for p in parts])  # noqa: E731
    h, w, t = given(stack("h")), given(stack("w")), given(stack("tokens"))
    gl, ge = given(stack("g_logp")), given(stack("g_entropy"))
    keep = torch.rand(S, N, V, generator=torch.Generator().manual_seed(1)) < 0.7
    keep[torch.arange(S)[:, None], torch.arange(N)[None], stack("tokens").long()] = True
    for shape in ((S, N, V), (S, 1, V), (1, N, V), (1, 1, V), (S, N, 1)):
        k = keep
        for dim, n in enumerate(shape):
            if n == 1:
                k = k.any(dim, keepdim=True)
        lp, ent, stats = nr.readout_score_with_stats(h, w, 1.0, given(k.to(torch.uint8)), t)
        gh, gw = nr.readout_score_grad(h, w, 1.0, given(k.to(torch.uint8)), t, stats, ent, gl, ge)
        for s, p in enumerate(parts):
            p.add = torch.where(k.expand(S, N, V)[s], 0.0, -math.inf).double()
            want, tol = p.want()
            for name, got in (("logp", lp), ("entropy", ent), ("grad_hidden", gh), ("grad_weight", gw)):
                agree(values(got)[s], want[name], tol[name], f"{shape} seed {s} {name}")


def test_one_gradient_alone():
    c = Case(30, 400, 48)
    both = c.run()
    h, w, t = given(c.h), given(c.w), given(c.tokens)
    lp, ent, stats = nr.readout_score_with_stats(h, w, c.tau, None, t)
    arg = (h, w, c.tau, None, t, stats, ent, given(c.g_logp), given(c.g_entropy))
    gh, none = nr.readout_score_grad(*arg, want_weight=False)
    assert none is None and np.array_equal(gh.to_numpy(), both["grad_hidden"].to_numpy())
    none, gw = nr.readout_score_grad(*arg, want_hidden=False)
    assert none is None and np.array_equal(gw.to_numpy(), both["grad_weight"].to_numpy())


def test_captured_calls_replay():
    """The forward and its backward as a graph, replayed over new inputs with eager calls between."""
    c = Case(90, 1000, 64, "bf16", "vd")
    h, w, t, gl, ge = (given(x) for x in (c.h, c.w, c.tokens, c.g_logp, c.g_entropy))
    rowf = lambda: nr.Tensor((c.rows,), "f32")  # noqa: E731
    lp, ent, base, rest, st = rowf(), rowf(), rowf(), rowf(), nr.Tensor((c.rows,), "u8")
    gh, gw = nr.Tensor((c.rows, c.d), "bf16"), nr.Tensor((c.V, c.d), "bf16")
    head = (h.ptr, w.ptr, nr.NT_BF16, nr.NT_READOUT_W_VD, c.rows, c.V, c.d, c.d, c.d, None, 0, nr.NT_MASK_NONE, 0, c.tau,
            t.ptr)
    a = nr.NtRlReadoutStatsArgs(*head, lp.ptr, ent.ptr, base.ptr, rest.ptr, st.ptr)
    b = nr.NtRlReadoutStatsGradArgs(*head, base.ptr, rest.ptr, ent.ptr, gl.ptr, ge.ptr, gh.ptr, gw.ptr, c.d, c.d)

    def calls():
        nr._check(nr.lib().nt_hip_rl_readout_score_stats(C.byref(a)), "stats")
        nr._check(nr.lib().nt_hip_rl_readout_score_backward(C.byref(b)), "backward")

    calls()
    nr.sync()
    g = Capture()
    with g:
        calls()
    for k in range(3):
        other = Case(90, 1000, 64, "bf16", "vd", seed=k + 1)
        want = other.run()  # eager, between the replays
        for dst, src in ((h, other.h), (w, other.w), (t, other.tokens), (gl, other.g_logp), (ge, other.g_entropy)):
            s = given(src)
            view = ops.Layout.contiguous(s.shape)
            ops.write(dst, view, s, view)
        g.replay()
        nr.sync()
        for name, got in (("logp", lp), ("entropy", ent), ("grad_hidden", gh), ("grad_weight", gw)):
            assert np.array_equal(got.to_numpy(), want[name].to_numpy()), (k, name)
    g.close()


def test_a_policy_step_with_an_8_bit_rollout():
    """Tokens drawn from the readout in 8 bits, then the policy loss on the readout's own log-probabilities and its
    gradients: through sample_logp, readout_score_with_stats, clipped_policy_loss and readout_score_grad."""
    S, B, T, V, d = 1, 4, 16, 1200, 64
    c = Case(S * B * T, V, d, "bf16", "vd", entropy=False)
    h, w = given(c.h), given(c.w)
    q, qs = ops.quantize_int8(h, ops.Layout.contiguous(h.shape))
    wq, ws = ops.quantize_int8(w, ops.Layout.contiguous(w.shape))
    logits = ops.matmul_int8(q, qs, wq, ws, "f32")
    # each logit: both operands off by half a step of their row's scale
    exact = c.h.double() @ c.w.double().t()
    hs, wss = values(qs)[:, None], values(ws)[None, :]
    bound = 0.5 * hs * c.w.double().abs().sum(1)[None, :] + 0.5 * wss * c.h.double().abs().sum(1)[:, None] + \
        0.25 * d * hs * wss
    assert ((values(logits) - exact).abs() <= bound * (1 + 1e-5)).all()
    ids, old, = nr.sample_logp(logits, 1.0, None, nr.Rng(3, "rollout"))
    c.tokens = torch.from_numpy(ids.to_numpy().astype(np.int32))
    hid = nr.Tensor((S, B, T, d), "bf16", h.buf)
    tok, old = nr.Tensor((S, B, T), "i32", ids.buf), nr.Tensor((S, B, T), "f32", old.buf)
    adv = given(torch.randn(S, B, generator=torch.Generator().manual_seed(2)))
    clip, red = nr.Clip.symmetric(0.2), nr.TokenReduction.TOKEN_MEAN
    lp, _, stats = nr.readout_score_with_stats(hid, w, 1.0, None, tok, entropy=False, layout="vd")
    loss = nr.clipped_policy_loss(lp, old, adv, None, clip, red)
    gl = nr.clipped_policy_loss_backward(lp, old, adv, None, clip, red)
    gh, gw = nr.readout_score_grad(hid, w, 1.0, None, tok, stats, g_logp=gl, layout="vd")
    assert np.isfinite(loss.to_numpy()).all() and gh.shape == hid.shape
    c.g_logp = values(gl).ravel().float()
    want, tol = c.want()
    agree(values(lp).ravel(), want["logp"], tol["logp"], "logp")
    agree(values(gh).reshape(c.rows, d), want["grad_hidden"], tol["grad_hidden"], "grad_hidden")
    agree(values(gw), want["grad_weight"], tol["grad_weight"], "grad_weight")


# Sizes that every tile, split and cut of the products is taken at: 256 x 256 tiles (300 x 32768, 1500 x 17001), those in
# whole rounds with a rest beside them (2100 x 32768), 128 x 128 and 64 x 128 ones, k split and not, in both layouts.
@pytest.mark.parametrize("rows,V,d,dtype,layout,mask", [
    (300, 32768, 512, "bf16", "dv", "none"), (1500, 17001, 520, "f16", "vd", "u8_shared"),
    (1500, 17001, 512, "bf16", "vd", "f32_shared"), (2100, 32768, 512, "bf16", "dv", "u8"),
    (2100, 32768, 512, "bf16", "dv", "f32_shared"), (2100, 32768, 520, "f16", "vd", "f32"),
    (2100, 16640, 1100, "bf16", "dv", "u8"), (2100, 16640, 1100, "f16", "vd", "none"), (2050, 17001, 1096, "bf16", "vd", "f32_shared"),
    (700, 9000, 200, "bf16", "vd", "f32"), (130, 30011, 520, "f16", "dv", "none"), (64, 20000, 300, "bf16", "dv", "none"),
    (65, 20000, 304, "bf16", "vd", "u8_shared"), (1, 50257, 128, "bf16", "vd", "none")])
def test_large_sizes(rows, V, d, dtype, layout, mask):
    c = Case(rows, V, d, dtype, layout, mask, tau=0.9)
    got = c.run()
    for name in ("h", "w", "tokens", "g_logp", "g_entropy", "add"):
        setattr(c, name, getattr(c, name).to("cuda"))
    device = torch.get_default_device()
    torch.set_default_device("cuda")
    try:
        want, tol = c.want()
    finally:
        torch.set_default_device(device)
    for k in got:
        agree(values(got[k]).to("cuda"), want[k], tol[k], k)
    if rows <= 512:  # the tokens' entries of G whole: the gradients are off by their own rounding and the other entries'
        u = HALF_STEP[dtype]
        for k in ("grad_hidden", "grad_weight"):
            off = (values(got[k]).to("cuda") - want[k]).norm() / want[k].norm()
            assert off <= 0.6 * u, (k, float(off))  # (a rounding alone: u / sqrt(3) at the most)


def test_a_padded_batch_holds_nothing_back():
    """Half the positions padded (upstream gradients zero, hidden states NaN, tokens -1): the others' results are those of
    the batch without them."""
    c = Case(96, 1000, 64, "bf16", "vd")
    pad = torch.arange(96) % 2 == 1
    c.h[pad], c.tokens[pad], c.g_logp[pad], c.g_entropy[pad] = math.nan, -1, 0.0, 0.0
    full = {k: values(v) for k, v in c.run(check=False).items()}
    d = Case(96, 1000, 64, "bf16", "vd")
    d.rows, d.h, d.tokens, d.g_logp, d.g_entropy = 48, c.h[~pad], c.tokens[~pad], c.g_logp[~pad], c.g_entropy[~pad]
    part = {k: values(v) for k, v in d.run().items()}
    for k in ("logp", "entropy", "base", "rest"):
        assert torch.equal(full[k][~pad], part[k]), k
    want, tol = d.want()
    agree(full["grad_hidden"][~pad], want["grad_hidden"], tol["grad_hidden"], "grad_hidden")
    agree(full["grad_weight"], want["grad_weight"], tol["grad_weight"], "grad_weight")
    assert (full["grad_hidden"][pad] == 0).all()


def test_the_same_token_at_every_position():
    c = Case(300, 700, 40, "bf16", "dv", tau=0.8)
    c.tokens[:] = 699
    check(c)


class Held:
    """A torch allocation as the buffer behind a tensor."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def test_offsets_past_32_bits():
    """A keep-mask of 4.8 GB and G in 19 pieces: the last rows and the first against the formulas."""
    R, V, d = 40000, 120001, 8
    c = Case(R, V, d, "bf16", "vd", entropy=False)
    g = torch.Generator(device="cuda").manual_seed(3)
    keep = torch.empty(R, V, dtype=torch.uint8, device="cuda").random_(0, 3, generator=g)  # a third excluded
    keep[torch.arange(R), c.tokens.long()] = 1
    torch.cuda.synchronize()
    m = nr.Tensor((R, V), "u8", Held(keep))
    h, w, t = given(c.h), given(c.w), given(c.tokens)
    lp, _, stats = nr.readout_score_with_stats(h, w, 1.0, m, t, entropy=False, layout="vd")
    gh, gw = nr.readout_score_grad(h, w, 1.0, m, t, stats, g_logp=given(c.g_logp), layout="vd")
    lp, gh, gw = values(lp), values(gh), values(gw)
    for at in (slice(0, 40), slice(R // 2, R // 2 + 40), slice(R - 40, R)):
        e = Case(40, V, d, "bf16", "vd", entropy=False)
        e.h, e.w, e.tokens, e.g_logp = c.h[at], c.w, c.tokens[at], c.g_logp[at]
        e.add = torch.where(keep[at].cpu() > 0, 0.0, -math.inf).double()
        want, tol = e.want()
        agree(lp[at], want["logp"], tol["logp"], "logp")
        agree(gh[at], want["grad_hidden"], tol["grad_hidden"], "grad_hidden")
    # a column's gradient from all rows, at both ends of the vocabulary
    W, H, at = c.w.double().cuda(), c.h.double().cuda(), c.tokens.long().cuda()
    gl = c.g_logp.double().cuda()
    cols = torch.tensor([0, 1, 65000, V - 2, V - 1], device="cuda")
    G = torch.zeros(R, 5, dtype=torch.float64, device="cuda")
    for r in range(0, R, 2000):
        s = slice(r, r + 2000)
        z = (H[s] @ W.t()).masked_fill_(keep[s] == 0, -math.inf)
        G[s] = -gl[s, None] * (z[:, cols] - torch.logsumexp(z, 1, keepdim=True)).exp()
    G += gl[:, None] * (at[:, None] == cols[None, :])
    want, size = G.t() @ H, G.abs().t() @ H.abs()
    u = HALF_STEP["bf16"]
    # (dp under 2^-12; each piece's sum of 40000 f32 terms)
    assert ((gw.cuda()[cols] - want).abs() <= (u + 2.0 ** -12 + R * 2.0 ** -24) * size + u * want.abs()).all()


# ----------------------------------------------------------------------------- far from zero

def exact_case(rows, V, d, dtype, layout, mask, tau, grid, seed=0):
    """A case whose logits are exact in f32 in any order of their sums: integers times multiples of `grid`, all held in
    the operands' type, and a temperature that is a power of two."""
    c = Case(rows, V, d, dtype, layout, mask, tau=tau, seed=seed)
    g = torch.Generator().manual_seed(seed + rows + V)
    c.h = torch.randint(-3, 4, (rows, d), generator=g).to(TORCH[dtype])
    w = (torch.randint(-250, 251, (V, d), generator=g).double() * grid).to(TORCH[dtype])
    c.w = w if layout == "vd" else w.t().contiguous()
    return c


def logits64(c):
    return c.h.double() @ (c.w.double().t() if c.layout == "vd" else c.w.double())


@pytest.mark.parametrize("bias", [-1e4, -65504.0, -1e9, torch.finfo(torch.float32).min, 1e9])
@pytest.mark.parametrize("rows,V,d,dtype,layout,kind", [(70, 1000, 8, "bf16", "dv", "f32"), (5, 640, 16, "f16", "vd", "f32_shared"),
                                                        (300, 33000, 24, "bf16", "vd", "f32_shared"),
                                                        (600, 5001, 8, "bf16", "dv", "bf16_bias")])
def test_a_large_bias_in_every_column(rows, V, d, dtype, layout, kind, bias):
    """tempered_logits' own f32 values, x / T + mask rounded once (the quotient is exact here), and the softmax of those:
    the same but for the base when the row's largest is taken off them."""
    c = exact_case(rows, V, d, dtype, layout, kind, 2.0, 2.0 ** -9)
    c.mask = torch.full_like(c.mask, max(bias, torch.finfo(c.mask.dtype).min))
    z = (logits64(c) / c.tau).float() + c.mask.float()  # f32
    assert z.isfinite().all()
    top = z.amax(1, keepdim=True)
    c.add = (z - top).double() - logits64(c) / c.tau
    got, (want, tol) = c.run(), c.want()
    assert torch.equal(values(got["base"]), top[:, 0].double())
    for k in ("logp", "rest", "entropy", "grad_hidden", "grad_weight"):
        agree(values(got[k]), want[k], tol[k], k)


@pytest.mark.parametrize("rows,V,d,dtype,layout,kind", [(70, 1000, 8, "bf16", "dv", "none"), (5, 640, 16, "f16", "vd", "u8"),
                                                        (520, 5000, 8, "bf16", "vd", "u8_shared"), (40, 901, 12, "bf16", "vd", "f32")])
def test_a_large_logit_in_every_column(rows, V, d, dtype, layout, kind):
    """2^17 added to every logit by a column of H and a row of W: the scores and the gradients of all other columns as
    without them."""
    c = exact_case(rows, V, d, dtype, layout, kind, 1.0, 2.0 ** -6)
    want, tol = c.want()
    one = torch.full((rows, 1), 256.0, dtype=c.h.dtype)
    row = torch.full((V, 1), 512.0, dtype=c.h.dtype)
    far = exact_case(rows, V, d, dtype, layout, kind, 1.0, 2.0 ** -6)
    far.h = torch.cat([one, c.h], 1)
    far.w = torch.cat([row, c.w], 1) if layout == "vd" else torch.cat([row.t(), c.w], 0)
    got = {k: values(v) for k, v in far.run().items()}
    assert torch.equal(got["base"], want["base"] + 2.0 ** 17)
    got["grad_hidden"] = got["grad_hidden"][:, 1:]
    got["grad_weight"] = got["grad_weight"][:, 1:] if layout == "vd" else got["grad_weight"][1:]
    for k in ("logp", "rest", "entropy", "grad_hidden", "grad_weight"):
        agree(got[k], want[k], tol[k], k)


@pytest.mark.parametrize("kind", ["none", "u8", "f32", "f32_shared"])
@pytest.mark.parametrize("layout", ["dv", "vd"])
@pytest.mark.parametrize("rows,V,d", [(75, 328, 40), (300, 1288, 72), (40, 264, 33)])
def test_row_padding_that_is_not_a_number(rows, V, d, layout, kind):
    """Aligned operands read in place, NaN behind the last value of each row: none of it reaches an output."""
    c = Case(rows, V, d, "bf16", layout, kind, tau=0.8)

    def padded(x):
        b = torch.full((x.shape[0], x.shape[1] + 8), math.nan, dtype=x.dtype)
        b[:, :x.shape[1]] = x
        return given(b), x.shape[1] + 8

    (h, ldh), (w, ldw) = padded(c.h), padded(c.w)
    m = None if c.mask is None else padded(c.mask) if c.mask.dtype == torch.float32 else (given(c.mask), V)
    kinds = {"n": nr.NT_MASK_NONE, "u": nr.NT_MASK_U8, "f": nr.NT_MASK_F32}
    t, gl, ge = given(c.tokens), given(c.g_logp), given(c.g_entropy)
    rowf = lambda: nr.Tensor((c.rows,), "f32")  # noqa: E731
    lp, ent, base, rest, st = rowf(), rowf(), rowf(), rowf(), nr.Tensor((c.rows,), "u8")
    lay = nr.NT_READOUT_W_DV if layout == "dv" else nr.NT_READOUT_W_VD
    head = (h.ptr, w.ptr, nr.NT_BF16, lay, c.rows, c.V, c.d, ldh, ldw, m[0].ptr if m else None,
            m[1] if m and c.mask.shape[0] > 1 else 0, kinds[kind[0]], 0, c.tau, t.ptr)
    a = nr.NtRlReadoutStatsArgs(*head, lp.ptr, ent.ptr, base.ptr, rest.ptr, st.ptr)
    nr._check(nr.lib().nt_hip_rl_readout_score_stats(C.byref(a)), "stats")
    gh, gw = nr.Tensor(tuple(c.h.shape), "bf16"), nr.Tensor(tuple(c.w.shape), "bf16")
    b = nr.NtRlReadoutStatsGradArgs(*head, base.ptr, rest.ptr, ent.ptr, gl.ptr, ge.ptr, gh.ptr, gw.ptr, c.d, c.w.shape[1])
    nr._check(nr.lib().nt_hip_rl_readout_score_backward(C.byref(b)), "backward")
    want, tol = c.want()
    for k, v in (("logp", lp), ("entropy", ent), ("base", base), ("rest", rest), ("grad_hidden", gh), ("grad_weight", gw)):
        agree(values(v), want[k], tol[k], k)


@pytest.mark.parametrize("layout", ["dv", "vd"])
@pytest.mark.parametrize("rows,V,d,spread", [(64, 400, 32, 20), (33, 1001, 45, 30), (600, 3001, 40, 20), (300, 9000, 72, 24)])
def test_f16_weight_gradients_of_rows_far_apart(rows, V, d, spread, layout):
    """Upstream gradients over many powers of two: the weight's gradient keeps each row's own bits. Besides G's rounding
    and its own, a value of H scaled next to the largest (2^15 at most, and over 2^14) is off by half a step of 2^-24
    where that leaves no more: 2^-39 of the largest |h| 2^e, times the row's G in its units of 2^e."""
    c = Case(rows, V, d, "f16", layout, entropy=False, scale=6.0)
    g = torch.Generator().manual_seed(rows)
    c.g_logp = (2.0 ** torch.linspace(-spread / 2, spread / 2, rows))[torch.randperm(rows, generator=g)].float()
    if rows == 64:
        c.h[5] *= 2.0 ** -8  # (a small row, and one past half of f16's range)
        c.h[7] *= 2.0 ** 4
    h = c.h.double()
    z = logits64(c) / c.tau
    dz = (d + 8) * 2.0 ** -24 * (h.abs() @ (c.w.double().abs().t() if layout == "vd" else c.w.double().abs())).amax(1, keepdim=True)
    p = torch.softmax(z, 1)
    gl = c.g_logp.double()[:, None]
    G = -gl * p
    G[torch.arange(rows), c.tokens.long()] += gl[:, 0]
    up = 2.0 ** (torch.floor(torch.log2(gl.abs())) + 1)
    u = HALF_STEP["f16"]
    dG = (u + 2.0 ** -22) * G.abs() + (4 * dz + 2.0 ** -20) * gl.abs() * p + 2.0 ** -38 * up
    want = h.t() @ G
    tol = h.abs().t() @ dG + rows * 2.0 ** -24 * (h.abs().t() @ G.abs()) + u * want.abs() + 2.0 ** -25
    tol = tol + 2.0 ** -39 * float((h.abs().amax(1, keepdim=True) * up).max()) * (G.abs() / up).sum(0)[None, :]
    # (an f16 of 65520 or more, half a step past the largest, is infinite; none is too near to tell)
    past = want.abs() - tol >= 65520.0
    assert (past | (want.abs() + tol < 65520.0)).all()
    want = torch.where(past, want.sign() * math.inf, want)
    if layout == "vd":
        want, tol = want.t(), tol.t()
    agree(values(c.run()["grad_weight"]), want, tol, "grad_weight")


@pytest.mark.parametrize("shape", [(0, 5, 300), (1, 5, 300), (300,), None])
def test_no_seeds(shape):
    """A weight of no seeds: empty results and gradients, with a mask and without."""
    h, w, t = nr.Tensor((0, 5, 16), "bf16"), nr.Tensor((0, 16, 300), "bf16"), nr.Tensor((0, 5), "i32")
    m = None if shape is None else nr.Tensor(shape, "u8")
    lp, ent, stats = nr.readout_score_with_stats(h, w, 1.0, m, t)
    gh, gw = nr.readout_score_grad(h, w, 1.0, m, t, stats, ent, lp, ent)
    assert lp.shape == ent.shape == (0, 5) and gh.shape == (0, 5, 16) and gw.shape == (0, 16, 300)


# Every tile, split k and unsplit, of each gradient's product (unsplit: dW, and dH of a DV weight, written as they are), and
# dW's columns in whole rounds with a rest beside them: what each takes is asserted in tests/test_tile_plan.py.
PLANS = [(520, 136, 40, "bf16", "dv", "f32"), (520, 130, 40, "f16", "vd", "none"), (1030, 130, 40, "bf16", "dv", "u8"),
         (520, 1003, 40, "f16", "vd", "none"), (4100, 130, 1001, "f16", "dv", "none"), (4100, 8200, 40, "bf16", "vd", "u8_shared"),
         (3000, 130, 4100, "bf16", "dv", "none"), (4100, 130, 4100, "f16", "dv", "f32_shared"), (520, 33000, 40, "bf16", "vd", "none"),
         (4100, 4100, 1001, "bf16", "vd", "none"), (4100, 4104, 1001, "f16", "dv", "none"), (520, 17001, 4100, "bf16", "vd", "none"),
         (520, 17008, 4100, "f16", "dv", "none")]
# A row's scores by 256 x 256 tiles, by 128 x 128 ones and by 64 x 128 ones (rows, and as few of them).
TILES_OF_ROWS = [(300, 32768, 512, 3), (130, 30016, 520, 3), (2100, 32768, 512, 300), (2100, 32768, 512, 130)]


@pytest.mark.parametrize("rows,V,d,dtype,layout,mask", PLANS)
def test_every_plan(rows, V, d, dtype, layout, mask):
    c = Case(rows, V, d, dtype, layout, mask, tau=0.9)
    got = c.run()
    for name in ("h", "w", "tokens", "g_logp", "g_entropy", "add"):
        setattr(c, name, getattr(c, name).to("cuda"))
    device = torch.get_default_device()
    torch.set_default_device("cuda")
    try:
        want, tol = c.want()
    finally:
        torch.set_default_device(device)
    for k in got:
        agree(values(got[k]).to("cuda"), want[k], tol[k], k)


@pytest.mark.parametrize("layout", ["dv", "vd"])
@pytest.mark.parametrize("rows,V,d,few", TILES_OF_ROWS)
def test_a_rows_scores_are_the_same_by_every_tile(rows, V, d, few, layout):
    c = Case(rows, V, d, "bf16", layout, "u8_shared", tau=0.7)
    h, w, m, t = given(c.h), given(c.w), given(c.mask), given(c.tokens)
    full = nr.readout_score_with_stats(h, w, c.tau, m, t, layout=layout)
    at = torch.linspace(0, rows - 1, few).long()
    part = nr.readout_score_with_stats(given(c.h[at]), w, c.tau, m, given(c.tokens[at]), layout=layout)
    for a, b in ((full[0], part[0]), (full[1], part[1]), (full[2].lse_base, part[2].lse_base), (full[2].lse_rest, part[2].lse_rest)):
        assert np.array_equal(a.to_numpy()[at.numpy()], b.to_numpy())


@pytest.mark.parametrize("dtype,layout", [("bf16", "dv"), ("bf16", "vd"), ("f16", "dv"), ("f16", "vd")])
@pytest.mark.parametrize("rows,V,d,live", [(700, 3001, 264, 700), (2100, 9000, 520, 2100), (2100, 9000, 520, 40), (5000, 40000, 72, 300),
                                           (130, 3001, 264, 7), (600, 70, 40, 600)])
def test_the_tokens_entries_are_whole_however_many_rows(rows, V, d, live, dtype, layout):
    """The gradients' error in norm: the written values' own rounding (a half step u at the most, u / sqrt(3) of it in
    the mean) and that of G's entries off the tokens, whatever the number of rows, of them those that something flows
    through, and a few upstream gradients far larger than the others. (dH of a DV weight past 512 rows: the part of it off
    the tokens, each row's by a factor within u of 1, u / sqrt(3) in the mean, besides.)"""
    c = Case(rows, V, d, dtype, layout, entropy=False)
    g = torch.Generator().manual_seed(rows + live)
    c.g_logp = torch.randn(rows, generator=g).exp() * (8.0 if dtype == "f16" else 1.0)
    c.g_logp[torch.randperm(rows, generator=g)[live:]] = 0.0
    got = {k: values(v).cuda() for k, v in c.run().items() if k.startswith("grad")}
    h, w = c.h.double().cuda(), c.w.double().cuda()
    w = w.t() if layout == "vd" else w
    gl = c.g_logp.double().cuda()[:, None]
    G = torch.softmax(h @ w, 1).mul_(-gl)
    G[torch.arange(rows, device="cuda"), c.tokens.long().cuda()] += gl[:, 0]
    gw = h.t() @ G
    for name, want in (("grad_hidden", G @ w.t()), ("grad_weight", gw if layout == "dv" else gw.t())):
        off = (got[name] - want).norm() / want.norm()
        most = 0.6
        if name == "grad_hidden" and layout == "dv" and rows > 512:
            others = G.clone()
            others[torch.arange(rows, device="cuda"), c.tokens.long().cuda()] = 0.0
            most += float((others @ w.t()).norm() / want.norm()) / math.sqrt(3)
        assert off <= most * HALF_STEP[dtype], (name, float(off) / HALF_STEP[dtype])


def test_every_row_has_one_of_two_tokens():
    """All rows in one 256 of the vocabulary, at each tile."""
    for rows, V, d, layout in ((9000, 400, 40, "vd"), (14000, 300, 520, "dv"), (30000, 256, 1032, "vd")):
        c = Case(rows, V, d, "bf16", layout, entropy=False)
        c.tokens[:] = V - 3
        c.tokens[::7] = V - 1
        got = c.run()
        for name in ("h", "w", "tokens", "g_logp", "g_entropy", "add"):
            setattr(c, name, getattr(c, name).to("cuda"))
        device = torch.get_default_device()
        torch.set_default_device("cuda")
        try:
            want, tol = c.want()
        finally:
            torch.set_default_device(device)
        for k in got:
            agree(values(got[k]).to("cuda"), want[k], tol[k], k)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,V,d", [(700, 3001, 264), (2100, 9000, 520)])
def test_rows_of_a_wide_weight_under_an_entropys_gradient(rows, V, d, dtype):
    """Rows of dH that are scaled for their token's entry, those whose entropy's gradient is too large for it and those of
    an entropy's gradient alone, where the token's entry is one of many: element by element, and in norm no worse than by
    both roundings."""
    c = Case(rows, V, d, dtype, "dv", "u8", tau=0.9)
    c.g_entropy = torch.randn(rows, generator=torch.Generator().manual_seed(1)) * c.g_logp.abs().mean() * \
        2.0 ** torch.randint(-8, 3, (rows,), generator=torch.Generator().manual_seed(2))
    c.g_logp[::3] = 0.0
    got = c.run()
    for name in ("h", "w", "tokens", "g_logp", "g_entropy", "add"):
        setattr(c, name, getattr(c, name).to("cuda"))
    device = torch.get_default_device()
    torch.set_default_device("cuda")
    try:
        want, tol = c.want()
    finally:
        torch.set_default_device(device)
    for k in got:
        agree(values(got[k]).to("cuda"), want[k], tol[k], k)
    for k in ("grad_hidden", "grad_weight"):
        off = (values(got[k]).to("cuda") - want[k]).norm() / want[k].norm()
        assert off <= 0.85 * HALF_STEP[dtype], (k, float(off) / HALF_STEP[dtype])  # (sqrt(0.6^2 + 1 / 3))


@pytest.mark.parametrize("rows,V,d,dtype,layout,mask", [(2100, 9000, 520, "bf16", "dv", "f32_shared"), (2100, 32768, 512, "bf16", "vd", "none"),
                                                        (333, 5003, 1001, "f16", "dv", "u8"), (4100, 70000, 72, "bf16", "dv", "none")])
def test_large_reruns_are_the_same_bytes(rows, V, d, dtype, layout, mask):
    c = Case(rows, V, d, dtype, layout, mask)
    a = {k: v.to_numpy() for k, v in c.run().items()}
    for _ in range(3):
        b = c.run()
        for k in a:
            assert np.array_equal(a[k], b[k].to_numpy()), k


@pytest.mark.skip(reason="faulted in a replay (illegal address), its cause not found: such calls are refused under capture")
def test_captured_calls_of_a_large_step_replay():
    """The same with 256 x 256 tiles, whole rounds and their rest, a mask and an entropy, replayed over other inputs."""
    R, V, d = 2100, 32768, 512
    c = Case(R, V, d, "bf16", "dv", "u8")
    bufs = [given(x) for x in (c.h, c.w, c.mask, c.tokens, c.g_logp, c.g_entropy)]
    h, w, m, t, gl, ge = bufs
    rowf = lambda: nr.Tensor((R,), "f32")  # noqa: E731
    lp, ent, base, rest, st = rowf(), rowf(), rowf(), rowf(), nr.Tensor((R,), "u8")
    gh, gw = nr.Tensor((R, d), "bf16"), nr.Tensor((d, V), "bf16")
    head = (h.ptr, w.ptr, nr.NT_BF16, nr.NT_READOUT_W_DV, R, V, d, d, V, m.ptr, V, nr.NT_MASK_U8, 0, c.tau, t.ptr)
    a = nr.NtRlReadoutStatsArgs(*head, lp.ptr, ent.ptr, base.ptr, rest.ptr, st.ptr)
    b = nr.NtRlReadoutStatsGradArgs(*head, base.ptr, rest.ptr, ent.ptr, gl.ptr, ge.ptr, gh.ptr, gw.ptr, d, V)

    def calls():
        nr._check(nr.lib().nt_hip_rl_readout_score_stats(C.byref(a)), "stats")
        nr._check(nr.lib().nt_hip_rl_readout_score_backward(C.byref(b)), "backward")

    calls()
    nr.sync()
    g = Capture()
    with g:
        calls()
    for k in range(3):
        other = Case(R, V, d, "bf16", "dv", "u8", seed=k + 1)
        want = other.run()  # eager, between the replays
        for dst, src in zip(bufs, (other.h, other.w, other.mask, other.tokens, other.g_logp, other.g_entropy)):
            s = given(src)
            view = ops.Layout.contiguous(s.shape)
            ops.write(dst, view, s, view)
        g.replay()
        nr.sync()
        for name, got in (("logp", lp), ("entropy", ent), ("grad_hidden", gh), ("grad_weight", gw)):
            assert np.array_equal(got.to_numpy(), want[name].to_numpy()), (k, name)
    g.close()


def test_a_step_too_large_for_capture_is_refused():
    """256 x 256 tiles, or scratch of 1 MiB and more, under stream capture: refused before anything is queued; the same
    calls run outside of one, and the next smaller step is captured."""
    for R, V, d, fits in ((2100, 32768, 512, False), (130, 30016, 64, False), (90, 1000, 64, True)):
        c = Case(R, V, d, "bf16", "vd")
        h, w, t, gl, ge = (given(x) for x in (c.h, c.w, c.tokens, c.g_logp, c.g_entropy))
        rowf = lambda: nr.Tensor((R,), "f32")  # noqa: E731
        lp, ent, base, rest, st = rowf(), rowf(), rowf(), rowf(), nr.Tensor((R,), "u8")
        gh, gw = nr.Tensor((R, d), "bf16"), nr.Tensor((V, d), "bf16")
        head = (h.ptr, w.ptr, nr.NT_BF16, nr.NT_READOUT_W_VD, R, V, d, d, d, None, 0, nr.NT_MASK_NONE, 0, c.tau, t.ptr)
        a = nr.NtRlReadoutStatsArgs(*head, lp.ptr, ent.ptr, base.ptr, rest.ptr, st.ptr)
        b = nr.NtRlReadoutStatsGradArgs(*head, base.ptr, rest.ptr, ent.ptr, gl.ptr, ge.ptr, gh.ptr, gw.ptr, d, d)
        L = nr.lib()
        assert L.nt_hip_rl_readout_score_stats(C.byref(a)) == 0 and L.nt_hip_rl_readout_score_backward(C.byref(b)) == 0
        nr.sync()
        g = Capture()
        with g:
            if fits:
                assert L.nt_hip_rl_readout_score_stats(C.byref(a)) == 0
            rc = L.nt_hip_rl_readout_score_backward(C.byref(b))
            text = L.nt_hip_last_error().decode()
        if fits:
            assert rc == 0 and g.nodes() > 5
        else:
            assert rc == -4 and "too large for stream capture" in text and g.nodes() == 0
        nr.sync()
        assert L.nt_hip_rl_readout_score_stats(C.byref(a)) == 0 and L.nt_hip_rl_readout_score_backward(C.byref(b)) == 0
        nr.sync()
        g.close()


@pytest.mark.parametrize("layout", ["dv", "vd"])
def test_padding_of_one_token(layout):
    """Most positions padded with one token, which live ones have too: the gradients of those that are not."""
    R, V, d = 3000, 5000, 264
    c = Case(R, V, d, "bf16", layout)
    pad = torch.rand(R, generator=torch.Generator().manual_seed(4)) < 0.9
    c.tokens[pad], c.g_logp[pad], c.g_entropy[pad] = 7, 0.0, 0.0
    live = (~pad).nonzero().ravel()
    c.tokens[live[::5]] = 7
    check(c)
