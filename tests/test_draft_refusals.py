"""Refusals of the drafted tokens' verification, the top log-probabilities and the distillation, before any device is
touched, and their argument structs' layouts."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import noetic_rl as nr

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = np.zeros(64, np.float32)
H = BUF.ctypes.data


def text():
    return nr.lib().nt_hip_last_error().decode()


def verify(**kw):
    a = dict(logits=H, draft_logits=H, dtype=0, seqs=2, drafted=1, vocab=4, ld=4, draft_ld=4, temperature=1.0, draft_temperature=1.0,
             tokens=H, uniforms=H, ids=H, accepted=H, logp=H, status=H)
    a.update(kw)
    return nr.lib().nt_hip_rl_verify_drafted(C.byref(nr.NtRlVerifyArgs(**a)))


@pytest.mark.parametrize("kw, said", [
    (dict(drafted=-1), "drafts"), (dict(drafted=128), "drafts"), (dict(seqs=-1), "sequences"), (dict(seqs=1 << 22), "positions"),
    (dict(vocab=0), "invalid rows"), (dict(ld=3), "invalid rows"), (dict(dtype=7), "invalid rows"), (dict(mask_kind=1), "mask null"),
    (dict(mask_kind=3, mask=H), "invalid rows"), (dict(mask_kind=1, mask=H, mask_ld=3), "mask_ld 3"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(draft_temperature=0.0), "draft temperature"), (dict(draft_temperature=float("inf")), "draft temperature"),
    (dict(draft_ld=3), "draft_ld"), (dict(vocab=1 << 31, ld=1 << 31, draft_ld=1 << 31), "vocab past"),
    (dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(uniforms=None), "null"), (dict(ids=None), "null"),
    (dict(accepted=None), "null"), (dict(status=None), "null"),
    (dict(mask_kind=1, mask=H, mask_rows=nr.NtMaskRows(3, 1, 0, 0)), "a multiple of"),
])
def test_verification_refuses(kw, said):
    assert verify(**kw) == -1 and said in text()


def top(**kw):
    a = dict(logits=H, dtype=0, rows=2, vocab=4, ld=4, temperature=1.0, k=2, ids=H, logp=H, status=H)
    a.update(kw)
    return nr.lib().nt_hip_rl_top_logprobs(C.byref(nr.NtRlTopArgs(**a)))


@pytest.mark.parametrize("kw, said", [
    (dict(k=0), "k 0"), (dict(k=5), "k 5 of 4"), (dict(k=1025, vocab=2000, ld=2000), "k 1025"), (dict(temperature=0.0), "temperature"),
    (dict(rows=1 << 24), "2^24"), (dict(vocab=1 << 31, ld=1 << 31), "2^31"), (dict(logits=None), "null"), (dict(ids=None), "null"),
    (dict(logp=None), "null"), (dict(status=None), "null"), (dict(mask_kind=2), "mask null"), (dict(dtype=-1), "dtype -1"),
])
def test_top_refuses(kw, said):
    assert top(**kw) == -1 and said in text()


def distill(**kw):
    a = dict(logits=H, dtype=0, rows=2, vocab=4, ld=4, temperature=1.0, k=2, ids=H, teacher_logp=H, loss=H, stats=H, status=H)
    a.update(kw)
    return nr.lib().nt_hip_rl_distill(C.byref(nr.NtRlDistillArgs(**a)))


def backward(**kw):
    a = dict(logits=H, dtype=0, rows=2, vocab=4, ld=4, temperature=1.0, k=2, ids=H, teacher_logp=H, stats=H, g_loss=H, grad=H, grad_ld=4)
    a.update(kw)
    return nr.lib().nt_hip_rl_distill_backward(C.byref(nr.NtRlDistillGradArgs(**a)))


SHARED = [(dict(k=0), "listed tokens"), (dict(k=1025), "listed tokens"), (dict(temperature=0.0), "temperature"), (dict(rows=1 << 24), "2^24"),
          (dict(vocab=1 << 31, ld=1 << 31, grad_ld=1 << 31), "2^31"), (dict(rows=1 << 23, vocab=1 << 20, ld=1 << 20, grad_ld=1 << 20), "2^24"),
          (dict(logits=None), "null"), (dict(ids=None), "null"), (dict(teacher_logp=None), "null"), (dict(stats=None), "null"),
          (dict(mask_kind=1), "mask null")]


@pytest.mark.parametrize("kw, said", SHARED + [(dict(tail=3), "tail 3"), (dict(tail=-1), "tail -1"), (dict(loss=None), "null"),
                                               (dict(status=None), "null")])
def test_distillation_refuses(kw, said):
    assert distill(**{k: v for k, v in kw.items() if k != "grad_ld"}) == -1 and said in text()


@pytest.mark.parametrize("kw, said", SHARED + [(dict(grad_dtype=3), "grad dtype"), (dict(grad_ld=3), "grad_ld"), (dict(g_loss=None), "null"),
                                               (dict(grad=None), "null")])
def test_its_backward_refuses(kw, said):
    assert backward(**kw) == -1 and said in text()


def test_null_arguments():
    for f in ("verify_drafted", "top_logprobs", "distill", "distill_backward"):
        assert getattr(nr.lib(), "nt_hip_rl_" + f)(None) == -1 and "null args" in text()


class Shape(nr.Tensor):
    """A tensor without memory, for checks that come before any."""

    def __init__(self, shape, dtype):
        class Nothing:
            ptr = 0
        super().__init__(shape, dtype, Nothing())


def test_the_mirrors_refuse():
    f32, i32 = lambda *s: Shape(s, "f32"), lambda *s: Shape(s, "i32")
    x = f32(2, 3, 8)
    ok = dict(uniforms=Shape((2, 3), "f64"))
    for args, kw, err, said in [
        ((x, None, i32(2, 2), -1.0, None, None), {}, ValueError, "temperature"),
        ((x, None, i32(2, 3), 1.0, None, None), ok, ValueError, "tokens"),
        ((x, None, f32(2, 2), 1.0, None, None), ok, ValueError, "tokens"),
        ((x, f32(2, 3, 8), i32(2, 2), 1.0, None, None), ok, ValueError, "draft logits"),
        ((x, Shape((2, 2, 8), "bf16"), i32(2, 2), 1.0, None, None), ok, TypeError, "f32 and bf16"),
        ((x, None, i32(2, 2), 1.0, None, None), {}, ValueError, "a stream is needed"),
        ((x, None, i32(2, 2), 1.0, None, None), dict(uniforms=Shape((2, 2), "f64")), ValueError, "uniforms"),
        ((x, None, i32(2, 2), 1.0, None, None), dict(ok, lengths=i32(3)), ValueError, "lengths"),
        ((x, None, i32(2, 2), 1.0, None, None), dict(ok, draft_temperature=0.0), ValueError, "draft temperature"),
        ((x, None, i32(2, 2), 1.0, Shape((3, 8), "u8"), None), ok, ValueError, "mask rank"),
        ((f32(8), None, i32(1), 1.0, None, None), ok, ValueError, "logits"),
    ]:
        with pytest.raises(err, match=said):
            nr.verify_drafted(*args, **kw)
    for k in (0, 9, 1025):
        with pytest.raises(ValueError, match="k"):
            nr.top_logprobs(x, k)
    for ids, lp, said in [(f32(2, 3, 4), f32(2, 3, 4), "ids"), (i32(2, 4), f32(2, 4), "ids"), (i32(2, 3, 0), f32(2, 3, 0), "ids"),
                          (i32(2, 3, 4), f32(2, 3, 5), "teacher"), (i32(2, 3, 4), i32(2, 3, 4), "teacher")]:
        with pytest.raises(ValueError, match=said):
            nr.distill_with_stats(x, ids, lp)
        with pytest.raises(ValueError, match=said):
            nr.distill_grad(x, ids, lp, nr.DistillStats(Shape((2, 3, 5), "f64")), f32(2, 3))
    with pytest.raises(ValueError, match="stats"):
        nr.distill_grad(x, i32(2, 3, 4), f32(2, 3, 4), nr.DistillStats(Shape((2, 2, 5), "f64")), f32(2, 3))
    with pytest.raises(ValueError, match="g_loss"):
        nr.distill_grad(x, i32(2, 3, 4), f32(2, 3, 4), nr.DistillStats(Shape((2, 3, 5), "f64")), f32(2))
    with pytest.raises(ValueError, match=r"\[S, B, T, V\]"):
        nr.distillation_loss(x, i32(2, 3, 4), f32(2, 3, 4))


def test_struct_layouts(tmp_path):
    body, names = [], ("NtRlVerifyArgs", "NtRlTopArgs", "NtRlDistillArgs", "NtRlDistillGradArgs")
    for n in names:
        body.append(f'printf("{n} %zu\\n", sizeof({n}));')
        body += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for f, _ in getattr(nr, n)._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"noetic_hip.h\"\nint main(void) {\n" + "\n".join(body) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for n in names:
        cls = getattr(nr, n)
        assert int(got[n]) == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(cls, f).offset
