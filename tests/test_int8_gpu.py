"""Rows in 8 bits and their product against the definitions in 64 bits: the integers and the scales are equal, the
products within their roundings (the integer sum to f32, two scalings: 3 half steps of 2^-24; the output type's half
step; f16's steps of 2^-24)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import noetic_ops as ops
import noetic_rl as nr
from tests.test_kept_blocks_gpu import Capture

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def device():
    nr.claim(0)
    yield


def given(t):
    name = {v: k for k, v in TORCH.items()}.get(t.dtype, "i8")
    t = t.contiguous()
    a = t.view(torch.int16).numpy().view(np.uint16) if name in ("bf16", "f16") else t.numpy()
    return nr.Tensor.from_numpy(a, name)


def quantized(x):
    """The definition: s = max |x| / 127 rounded to f32, q = round(x / s), ties to even, of the exact quotient (64 bits
    tell every f32 quotient from a half: they differ by 2^-33 at least)."""
    x = x.double()
    bad = ~x.isfinite().all(-1)
    s = (x.abs().amax(-1) / 127.0).float() if x.shape[-1] else torch.zeros(x.shape[:-1])
    q = torch.round(x / s.double()[..., None]).nan_to_num(0.0).clamp(-127, 127)
    q[(s == 0) | bad] = 0
    s[bad] = math.nan
    return q.to(torch.int8), s


def same(q, s, want):
    assert np.array_equal(q.to_numpy(), want[0].numpy())
    assert np.array_equal(s.to_numpy(), want[1].numpy(), equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (64, 64), (65, 130), (7, 1000), (300, 257), (2, 40000),
                                       (1, 16384), (4097, 24)])
def test_rows_and_columns(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 7 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))).to(TORCH[dtype])
    t = given(x)
    view = ops.Layout.contiguous(x.shape)
    q, s = ops.quantize_int8(t, view)
    same(q, s, quantized(x))
    for to in TORCH:
        back = ops.dequantize_int8(q, s, to)
        want = (quantized(x)[0].float() * quantized(x)[1][:, None]).to(TORCH[to])
        assert np.array_equal(back.to_f64(), want.double().numpy(), equal_nan=True)  # (f16 rows past its range: NaN)
    q, s = ops.quantize_int8(t, view.swapped(0, 1))
    assert q.shape == (cols, rows) and s.shape == (cols,)
    same(q, s, quantized(x.t()))


@pytest.mark.parametrize("n,cols", [(256, 1), (257, 1), (511, 65), (513, 64), (1500, 700), (4099, 130), (70001, 3),
                                    (300, 16400), (515, 16321), (260, 16319)])
def test_long_columns(n, cols):
    """Columns of one workgroup and of several, at the borders between them: a column's largest value, its NaN or its
    infinity in the first part, the last, or alone in the last row."""
    g = torch.Generator().manual_seed(n + cols)
    x = torch.randn(n, cols, generator=g)
    x[n - 1] *= 100.0
    x[n // 2, ::3] *= 1000.0
    x[:, 0] = 0.0
    x[n - 1, 0] = -1e-30
    if cols > 2:
        x[n - 1, 1] = math.nan
        x[0, 2] = -math.inf
    for dtype in TORCH.values():
        y = x.to(dtype)
        q, s = ops.quantize_int8(given(y), ops.Layout([cols, n], [1, cols]))
        same(q, s, quantized(y.t()))


def test_borders():
    """Quotients at and next to halves: rows whose largest value is 127 times a power of two or three of it, so that
    the scale and the halves are exact, and each half's neighbours in f32."""
    for unit in (1.0, 2.0 ** -40, 3.0, 2.0 ** -130, 2.0 ** 100):
        half = (torch.arange(-126, 126).double() + 0.5) * unit
        h = half.float()
        x = torch.cat([torch.tensor([127.0 * unit], dtype=torch.float64).float(), h,
                       torch.nextafter(h, torch.tensor(math.inf)), torch.nextafter(h, torch.tensor(-math.inf))])[None]
        q, s = ops.quantize_int8(given(x), ops.Layout.contiguous(x.shape))
        same(q, s, quantized(x))
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2000, 500, generator=g)
    x = x * (torch.rand(2000, 1, generator=g) + 0.5)
    s = quantized(x)[1].double()[:, None]
    near = ((torch.round(x.double() / s - 0.5) + 0.5) * s).float()  # the f32 values nearest to halves
    near[:, 0] = x.abs().amax(1)
    q, s = ops.quantize_int8(given(near), ops.Layout.contiguous(near.shape))
    same(q, s, quantized(near))


def test_rows_that_are_not_plain():
    tiny = 2.0 ** -149
    x = torch.zeros(9, 20)
    x[1, 3] = math.nan
    x[2, 4] = -math.inf
    x[3] = tiny
    x[4] = 100 * tiny * torch.linspace(-1, 1, 20)
    x[5] = 1000 * tiny * torch.linspace(-1, 1, 20)
    x[6] = 3.4e38 * torch.linspace(-1, 1, 20)
    x[7, 0] = -0.0
    x[8] = -5.0
    for t in (x, x.t().contiguous().t()):
        view = ops.Layout.contiguous(x.shape) if t.is_contiguous() else ops.Layout([9, 20], [1, 9])
        q, s = ops.quantize_int8(given(t if t.is_contiguous() else t.t()), view)
        same(q, s, quantized(x))


def test_views():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 6, 10, generator=g)
    t, full = given(x), ops.Layout.contiguous(x.shape)
    for view, want in ((full, x), (full.swapped(0, 1), x.transpose(0, 1)), (full.swapped(1, 2), x.transpose(1, 2)),
                       (full.swapped(0, 2), x.transpose(0, 2)), (full.narrowed([range(1, 3), range(2, 6), range(3, 8)]),
                                                                 x[1:3, 2:6, 3:8]),
                       (ops.Layout([10], [0], 5), x.flatten()[5].expand(10)), (ops.Layout([60, 2, 2], [4, 2, 1]), x.reshape(60, 2, 2)),
                       (ops.Layout([3, 10], [0, 1], 20), x.flatten()[20:30].expand(3, 10))):
        q, s = ops.quantize_int8(t, view)
        same(q, s, quantized(want.contiguous()))
    for shape in ((0, 5), (5, 0), (0, 0)):
        q, s = ops.quantize_int8(given(torch.zeros(1)), ops.Layout(shape))
        assert q.shape == shape and (s.to_numpy() == 0).all()
        assert ops.dequantize_int8(q, s).shape == shape


def product(a, sa, b, sb):
    return (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None, :]


def agree(got, want, dtype):
    off = (torch.from_numpy(got.to_f64()) - want).abs()
    step = torch.finfo(TORCH[dtype]).eps / 2 if dtype != "f32" else 0.0
    tol = want.abs() * (4 * 2.0 ** -24 + step) + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert (off <= tol).all(), f"{(off - tol).max():.3g}"


PRODUCTS = [(1, 1, 1), (1, 5, 16), (2, 300, 48), (16, 64, 64), (33, 100, 77), (64, 1000, 128), (65, 257, 1000),
            (128, 128, 4096), (300, 520, 208), (257, 255, 33), (1, 4099, 512), (5, 40, 20000), (700, 31, 96),
            # every tile and a split k; up to four rows beside five
            (6, 276, 12096), (100, 152, 10496), (3, 33, 1040), (4, 1001, 2064), (5, 1001, 2064), (600, 5000, 272),
            (2049, 4100, 96), (70, 33000, 64)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products(m, n, k, dtype):
    g = torch.Generator().manual_seed(m + 1000 * n + k)
    a, b = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    sa, sb = torch.rand(m, generator=g) * 1e-3, torch.rand(n, generator=g) * 1e-2
    y = ops.matmul_int8(given(a), given(sa), given(b), given(sb), dtype)
    assert y.shape == (m, n)
    agree(y, product(a, sa, b, sb), dtype)


# Every tile, split k and not, with sides that end inside one: what each takes is asserted in tests/test_tile_plan.py. (5 to
# 64 rows against a few columns are 1 to 16 tiles, whose k is split into 512 bytes and more.)
PLANS = [(5, 40, 48), (5, 40, 2064), (64, 1000, 8192), (17, 500, 1040), (600, 40, 131071), (1000, 4100, 48), (3001, 4100, 300),
         (1000, 4100, 10496)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", PLANS)
def test_every_plan(m, n, k, dtype):
    g = torch.Generator().manual_seed(m + 1000 * n + k)
    a, b = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    sa, sb = torch.rand(m, generator=g) * 1e-3, torch.rand(n, generator=g) * 1e-2
    y = ops.matmul_int8(given(a), given(sa), given(b), given(sb), dtype)
    agree(y, product(a, sa, b, sb), dtype)


def test_sums_at_their_ends():
    """All of one sign at the largest k: the sums reach 2^31 - 2^14 and its negative, -128 among the values."""
    k = 131071
    a = torch.full((3, k), -128, dtype=torch.int8)
    b = torch.full((2, k), -128, dtype=torch.int8)
    b[1] = 127
    one = torch.ones(3)
    y = ops.matmul_int8(given(a), given(one), given(b), given(one[:2].contiguous()))
    assert y.to_numpy()[0].tolist() == [float(np.float32(16384 * k)), float(np.float32(-128 * 127 * k))]


def test_scales_that_are_not_plain():
    """A NaN scale (a row that held a NaN) makes its outputs NaN and no others; zero scales zeros; k = 0 zeros."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(5, 40, generator=g)
    x[2, 7], x[3] = math.nan, 0.0
    q, s = ops.quantize_int8(given(x), ops.Layout.contiguous(x.shape))
    w = torch.randn(70, 40, generator=g)
    wq, ws = ops.quantize_int8(given(w), ops.Layout.contiguous(w.shape))
    y = ops.matmul_int8(q, s, wq, ws).to_numpy()
    assert np.isnan(y[2]).all() and (y[3] == 0).all() and np.isfinite(y[[0, 1, 3, 4]]).all()
    y = ops.matmul_int8(nr.Tensor((2, 0), "i8"), given(torch.ones(2)), nr.Tensor((3, 0), "i8"), given(torch.ones(3)))
    assert (y.to_numpy() == 0).all()
    y = ops.matmul_int8(nr.Tensor((70, 0), "i8"), given(torch.ones(70)), nr.Tensor((300, 0), "i8"), given(torch.ones(300)))
    assert (y.to_numpy() == 0).all()
    assert ops.matmul_int8(nr.Tensor((0, 4), "i8"), nr.Tensor((0,), "f32"), nr.Tensor((3, 4), "i8"),
                           given(torch.ones(3))).shape == (0, 3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_leading_dimensions(dtype):
    """Operands and output inside larger buffers at odd places; the padding stays as it was."""
    m, n, k = 70, 90, 50
    g = torch.Generator().manual_seed(8)
    a, b = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    sa, sb = torch.rand(m, generator=g), torch.rand(n, generator=g)
    for shift, pad in ((1, 3), (16, 14), (0, 14)):
        A, B = (torch.full((r * (k + pad) + shift,), 99, dtype=torch.int8) for r in (m, n))
        A[shift:].view(m, k + pad)[:, :k], B[shift:].view(n, k + pad)[:, :k] = a, b
        out = torch.full((m * (n + pad) + shift,), 5.0).to(TORCH[dtype])
        ta, tb, to, tsa, tsb = given(A), given(B), given(out), given(sa), given(sb)
        es = 4 if dtype == "f32" else 2
        nr._check(nr.lib().nt_hip_matmul_int8(ta.ptr + shift, k + pad, tsa.ptr, tb.ptr + shift, k + pad, tsb.ptr, m, n, k,
                                              ops._DT[dtype], to.ptr + es * shift, n + pad), "matmul_int8")
        y = torch.from_numpy(to.to_f64())
        assert (y[:shift] == 5).all()
        y = y[shift:].view(m, n + pad)
        assert (y[:, n:] == 5).all()
        want = product(a, sa, b, sb)
        step = 4 * 2.0 ** -24 + (torch.finfo(TORCH[dtype]).eps / 2 if dtype != "f32" else 0.0)
        assert ((y[:, :n] - want).abs() <= want.abs() * step).all()
    y = ops.matmul_int8(given(a.view(7, 10, k)), given(sa.view(7, 10)), given(b), given(sb), dtype)
    assert y.shape == (7, 10, n)
    agree(nr.Tensor((m, n), dtype, y.buf), product(a, sa, b, sb), dtype)


@pytest.mark.parametrize("m", [1, 4, 5, 70, 300])
def test_no_k_at_any_stride(m):
    """k = 0: zeros, whatever the operands' addresses and strides."""
    n = 300
    sa, sb, out = given(torch.rand(m)), given(torch.rand(n)), given(torch.full((m, n), 5.0))
    for lda, ldb, at in ((0, 0, 0), (5, 16, 0), (16, 7, 0), (3, 1, 1), (64, 64, 8)):
        some = nr.Tensor((64,), "i8")
        nr._check(nr.lib().nt_hip_matmul_int8(some.ptr + at, lda, sa.ptr, some.ptr + at, ldb, sb.ptr, m, n, 0, 0, out.ptr, n),
                  "matmul_int8")
        assert (out.to_numpy() == 0).all()
        nr._check(nr.lib().nt_hip_matmul_int8(None, lda, sa.ptr, None, ldb, sb.ptr, m, n, 0, 0, out.ptr, n), "matmul_int8")
        assert (out.to_numpy() == 0).all()


def test_captured_calls_replay():
    m, n, k = 33, 500, 100
    g = torch.Generator().manual_seed(9)
    w = torch.randn(n, k, generator=g)
    wq, ws = ops.quantize_int8(given(w), ops.Layout.contiguous(w.shape))
    x, q, s, y = nr.Tensor((m, k), "f32"), nr.Tensor((m, k), "i8"), nr.Tensor((m,), "f32"), nr.Tensor((m, n), "f32")
    lay = ops.Layout.contiguous((m, k)).c()
    L = nr.lib()

    def calls():
        nr._check(L.nt_hip_quantize_int8(x.ptr, C.byref(lay), 0, q.ptr, s.ptr), "quantize")
        nr._check(L.nt_hip_matmul_int8(q.ptr, k, s.ptr, wq.ptr, k, ws.ptr, m, n, k, 0, y.ptr, n), "matmul")

    calls()
    nr.sync()
    cap = Capture()
    with cap:
        calls()
    for _ in range(3):
        xs = given(torch.randn(m, k, generator=g))
        view = ops.Layout.contiguous((m, k))
        ops.write(x, view, xs, view)
        eq, es = ops.quantize_int8(xs, view)
        want = ops.matmul_int8(eq, es, wq, ws).to_numpy()
        cap.replay()
        nr.sync()
        assert np.array_equal(y.to_numpy(), want)
    cap.close()


def test_a_product_with_much_scratch_is_refused_under_capture():
    """k of no whole chunks against a weight of 1.1 MB, whose copy is scratch: refused under stream capture before
    anything is queued, and right outside of one."""
    m, n, k = 8, 1100, 1001
    g = torch.Generator().manual_seed(5)
    a, b = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    sa, sb = torch.rand(m, generator=g), torch.rand(n, generator=g)
    ta, tb, tsa, tsb, y = given(a), given(b), given(sa), given(sb), nr.Tensor((m, n), "f32")
    call = lambda: nr.lib().nt_hip_matmul_int8(ta.ptr, k, tsa.ptr, tb.ptr, k, tsb.ptr, m, n, k, 0, y.ptr, n)  # noqa: E731
    nr.sync()
    cap = Capture()
    with cap:
        rc = call()
        text = nr.lib().nt_hip_last_error().decode()
    assert rc == -4 and "under stream capture" in text and cap.nodes() == 0
    cap.close()
    assert call() == 0
    agree(y, product(a, sa, b, sb), "f32")
    x = given(torch.randn(70, 70, 70, generator=g))  # (a view that is neither rows nor columns: its copy is scratch)
    lay, q, s = ops.Layout.contiguous((70, 70, 70)).swapped(0, 2).c(), nr.Tensor((70, 70, 70), "i8"), nr.Tensor((70, 70), "f32")
    quantize = lambda: nr.lib().nt_hip_quantize_int8(x.ptr, C.byref(lay), 0, q.ptr, s.ptr)  # noqa: E731
    nr.sync()
    cap = Capture()
    with cap:
        rc = quantize()
    assert rc == -4 and cap.nodes() == 0
    cap.close()
    assert quantize() == 0
