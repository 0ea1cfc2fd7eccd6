"""CPU tests of the training readout's and the 8-bit operators' refusals: arguments are checked before the device."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

import noetic_ops as ops
import noetic_rl as nr

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = np.zeros(4096, np.float32)
P = (BUF.ctypes.data + 63) // 64 * 64

STATS = dict(hidden=P, weight=P, dtype=nr.NT_BF16, layout=nr.NT_READOUT_W_VD, rows=4, vocab=32, dim=16, ldh=16, ldw=16,
             mask_kind=nr.NT_MASK_NONE, temperature=1.0, tokens=P, logp=P, status=P)
GRAD = {k: v for k, v in STATS.items() if k not in ("logp", "status")}
GRAD.update(lse_base=P, lse_rest=P, g_logp=P, grad_hidden=P, grad_weight=P, grad_hidden_ld=16, grad_weight_ld=16)


def refused(fn, *a):
    assert fn(*a) == -1
    return nr.lib().nt_hip_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(dtype=nr.NT_F32), "dtype 0"), (dict(layout=2), "layout 2"), (dict(rows=-1), "rows -1"),
    (dict(rows=(1 << 24) + 1), "at most 2^24"), (dict(vocab=0), "vocab 0"), (dict(vocab=(1 << 20) + 1), "1 to 2^20"),
    (dict(dim=0), "dim 0"), (dict(dim=65537, ldh=65537, ldw=65537), "1 to 65536"), (dict(ldh=15), "ldh 15"),
    (dict(ldw=15), "ldw 15"), (dict(ldw=(1 << 21) + 1), "at most 2^21"),
    (dict(layout=nr.NT_READOUT_W_DV, ldw=31), "ldw 31"), (dict(mask_kind=3, mask=P), "mask kind 3"),
    (dict(mask_kind=nr.NT_MASK_U8), "disagree"), (dict(mask=P), "disagree"),
    (dict(mask_kind=nr.NT_MASK_U8, mask=P, mask_ld=31), "mask_ld 31"),
    (dict(mask_kind=nr.NT_MASK_F32, mask=P + 2, mask_ld=32), "unaligned mask"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=math.inf), "temperature"),
    (dict(temperature=math.nan), "temperature"), (dict(temperature=1e-300), "temperature"), (dict(hidden=None), "null"),
    (dict(weight=None), "null"), (dict(tokens=None), "null"), (dict(hidden=P + 1), "unaligned"), (dict(weight=P + 1), "unaligned"),
])
def test_readout_refusals(change, text):
    L = nr.lib()
    assert text in refused(L.nt_hip_rl_readout_score_stats, C.byref(nr.NtRlReadoutStatsArgs(**dict(STATS, **change))))
    assert text in refused(L.nt_hip_rl_readout_score_backward, C.byref(nr.NtRlReadoutStatsGradArgs(**dict(GRAD, **change))))


def test_readout_outputs_are_checked():
    L = nr.lib()
    for change in (dict(logp=None), dict(status=None)):
        assert "null logp" in refused(L.nt_hip_rl_readout_score_stats, C.byref(nr.NtRlReadoutStatsArgs(**dict(STATS, **change))))
    for change, text in ((dict(grad_hidden=None, grad_weight=None), "no gradient"), (dict(grad_hidden_ld=15), "stride"),
                         (dict(grad_weight_ld=15), "stride"), (dict(grad_weight=P + 1), "unaligned"),
                         (dict(lse_base=None), "null lse_base"), (dict(lse_rest=None), "null lse_base"),
                         (dict(g_entropy=P), "without the entropy")):
        assert text in refused(L.nt_hip_rl_readout_score_backward, C.byref(nr.NtRlReadoutStatsGradArgs(**dict(GRAD, **change))))
    assert "null args" in refused(L.nt_hip_rl_readout_score_stats, None)
    assert "null args" in refused(L.nt_hip_rl_readout_score_backward, None)


def test_int8_refusals():
    L = nr.lib()
    lay = ops.Layout([4, 8]).c()
    assert "rank" in refused(L.nt_hip_quantize_int8, P, C.byref(ops.Layout([]).c()), 0, P, P)
    assert "rank" in refused(L.nt_hip_quantize_int8, P, None, 0, P, P)
    assert "dtype 5" in refused(L.nt_hip_quantize_int8, P, C.byref(lay), 5, P, P)
    assert "negative" in refused(L.nt_hip_quantize_int8, P, C.byref(ops.Layout([4, 8], [8, -1]).c()), 0, P, P)
    for hole in range(3):
        a = [P, P, P]
        a[hole] = None
        assert "null" in refused(L.nt_hip_quantize_int8, a[0], C.byref(lay), 0, a[1], a[2])
        assert "null" in refused(L.nt_hip_dequantize_int8, a[0], a[1], 4, 8, 0, a[2])
    assert "dtype 3" in refused(L.nt_hip_dequantize_int8, P, P, 4, 8, 3, P)
    assert "rows" in refused(L.nt_hip_dequantize_int8, P, P, -4, 8, 0, P)
    ok = dict(a=P, lda=16, a_scale=P, b=P, ldb=16, b_scale=P, m=4, n=8, k=16, dtype=0, out=P, ldo=8)
    for change, text in ((dict(dtype=4), "dtype 4"), (dict(m=-1), "[-1, 16]"), (dict(k=131072, lda=131072, ldb=131072), "131071"),
                         (dict(lda=15), "strides"), (dict(ldb=15), "strides"), (dict(ldo=7), "strides"),
                         (dict(lda=(1 << 22) + 1), "2^22"), (dict(m=1 << 24, n=1 << 24, ldo=1 << 24), "outputs"),
                         (dict(a=None), "null"), (dict(b_scale=None), "null"), (dict(out=None), "null"), (dict(out=P + 2), "unaligned")):
        assert text in refused(L.nt_hip_matmul_int8, *dict(ok, **change).values()), change


class Fake(nr.Tensor):
    """A tensor with no device behind it: what is refused never reads one."""

    def __init__(self, shape, dtype):
        class NoMemory:
            ptr = 0
        super().__init__(shape, dtype, NoMemory())


def test_mirror_refusals():
    h, w, t = Fake((6, 16), "bf16"), Fake((16, 32), "bf16"), Fake((6,), "i32")
    stats = nr.RowStats(Fake((6,), "f32"), Fake((6,), "f32"))
    with pytest.raises(ValueError, match="MatmulPrecision::Half"):
        nr.readout_score_with_stats(h, w, 1.0, None, t)
    with nr.matmul_precision_scope(nr.MatmulPrecision.HALF):
        for err, text, a in ((ValueError, "temperature", (h, w, 0.0, None, t)), (ValueError, "layout", (h, w, 1.0, None, t, True, "xy")),
                             (ValueError, "bf16 or f16 weight", (h, Fake((16, 32), "f32"), 1.0, None, t)),
                             (ValueError, "d 16 against the weight's 32", (h, w, 1.0, None, t, True, "vd")),
                             (nr.DTypeError, "casts are explicit", (Fake((6, 16), "f16"), w, 1.0, None, t)),
                             (ValueError, "seeds", (h, Fake((2, 16, 32), "bf16"), 1.0, None, t)),
                             (ValueError, "tokens shape", (h, w, 1.0, None, Fake((5,), "i32"))),
                             (ValueError, "tokens shape", (h, w, 1.0, None, Fake((6,), "f32"))),
                             (ValueError, "vocabulary mask of dtype", (h, w, 1.0, Fake((6, 32), "i32"), t)),
                             (ValueError, "does not broadcast", (h, w, 1.0, Fake((5, 32), "u8"), t))):
            with pytest.raises(err, match=text):
                nr.readout_score_with_stats(*a)
        with pytest.raises(ValueError, match="no gradient"):
            nr.readout_score_grad(h, w, 1.0, None, t, stats, want_hidden=False, want_weight=False)
        with pytest.raises(ValueError, match="needs the forward's entropy"):
            nr.readout_score_grad(h, w, 1.0, None, t, stats, g_entropy=Fake((6,), "f32"))
        with pytest.raises(ValueError, match="g_logp: 5 values for 6 rows"):
            nr.readout_score_grad(h, w, 1.0, None, t, stats, g_logp=Fake((5,), "f32"))
    q, s = Fake((6, 16), "i8"), Fake((6,), "f32")
    with pytest.raises(TypeError, match="quantize_int8 of i32"):
        ops.quantize_int8(t, ops.Layout([6]))
    with pytest.raises(ValueError, match="rank 1"):
        ops.quantize_int8(h, ops.Layout([]))
    with pytest.raises(IndexError, match="leaves the buffer"):
        ops.quantize_int8(h, ops.Layout([6, 17]))
    with pytest.raises(ValueError, match="scales for the rows"):
        ops.dequantize_int8(q, Fake((5,), "f32"))
    with pytest.raises(TypeError, match="into i32"):
        ops.dequantize_int8(q, s, "i32")
    with pytest.raises(ValueError, match="matmul_int8"):
        ops.matmul_int8(q, s, Fake((8, 15), "i8"), Fake((8,), "f32"))
    with pytest.raises(TypeError, match="i8 and f32"):
        ops.matmul_int8(Fake((6, 16), "u8"), s, q, s)


@pytest.mark.parametrize("rows,scales", [(2, 100), (100, 2), (0, 1), (1, 0)])
def test_scales_of_rows_without_elements_are_counted(rows, scales):
    """Rows of no elements have a scale each: another number of them is refused, on either side of the product."""
    q, s = Fake((rows, 0), "i8"), Fake((scales,), "f32")
    other, one = Fake((3, 0), "i8"), Fake((3,), "f32")
    for call in (lambda: ops.dequantize_int8(q, s), lambda: ops.matmul_int8(q, s, other, one),
                 lambda: ops.matmul_int8(other, one, q, s)):
        with pytest.raises(ValueError, match="scales for the rows"):
            call()


@pytest.mark.parametrize("shape", [(0, 5, 32), (1, 5, 32), (0, 1, 32), (1, 1, 32), (32,)])
def test_masks_of_no_seeds(shape):
    """No seeds, a mask: shapes that broadcast are taken, others refused."""
    kind, mask, _, _ = nr._readout_vocab_mask(Fake(shape, "u8"), (0, 5, 32), 0, 32, 0)
    assert kind == nr.NT_MASK_U8 and mask.shape == shape
    with pytest.raises(ValueError, match="does not broadcast"):
        nr._readout_vocab_mask(Fake((2, 5, 32), "u8"), (0, 5, 32), 0, 32, 0)


def test_argument_struct_layouts_match_the_header(tmp_path):
    names = ("NtRlReadoutStatsArgs", "NtRlReadoutStatsGradArgs")
    lines = []
    for n in names:
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f[0]} %zu\\n", offsetof({n}, {f[0]}));' for f in getattr(nr, n)._fields_]
    c = tmp_path / "layout.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "noetic_hip.h"\nint main(void) {\n' + "\n".join(lines)
                 + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for n in names:
        cls = getattr(nr, n)
        assert int(got[n]) == C.sizeof(cls)
        for f in cls._fields_:
            assert int(got[f"{n}.{f[0]}"]) == getattr(cls, f[0]).offset, (n, f[0])
