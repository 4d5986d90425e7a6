"""8-bit integers with a scale a row on the GPU: quantisation code for code, the products against exact sums.

A product's bound: the sum is exact; three roundings in fp32 (the sum's, the two scales'), one to the result's type."""
import threading

import numpy as np
import pytest

from tests import more_ref as ref
from c0ven_amd._lib import MOE_ERROR
from tests.harness import moe
from tests.ops_dev import TYPES, Raw, decode, encode, hip

pytestmark = pytest.mark.gpu

TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step of the smallest values


def say(*a):
    print(*a, flush=True)


def room(*shape):
    return hip.full(shape, 0xA5, np.uint8)


def matrix(rows, cols, codes=None, scales=None):
    """An I8Matrix with a guard row behind it, and its buffers."""
    c, s = hip.full((rows + 1, ref.pad128(cols)), 0x5A, np.int8), hip.full(rows + 1, 7.0)
    if codes is not None:
        c.put(ref.i8_padded(codes))
        s.put(np.asarray(scales, np.float32))
    return moe.I8Matrix(c.ptr, s.ptr, rows, cols), c, s


def special(rows, cols, seed):
    """Normal rows of different sizes, with halves between codes and values a unit off them, empty and tiny rows, infinities, NaNs."""
    r = np.random.default_rng(seed)
    x = (r.normal(size=(rows, cols)) * np.exp2(r.integers(-20, 14, size=(rows, 1)))).astype(np.float32)
    for i in range(0, rows, 3):
        s = np.float32(2.0 ** float(r.integers(-8, 6)) * r.choice([1.0, 1.25, 1 + 2.0 ** -20]))
        x[i] = (r.integers(-127, 127, size=cols) + np.float32(0.5)) * s
        off = r.random(cols)
        x[i] = np.where(off < 0.3, np.nextafter(x[i], np.float32(np.inf)), np.where(off < 0.6, np.nextafter(x[i], np.float32(0)), x[i]))
        x[i, r.integers(cols)] = 127 * s
    for i, bad in enumerate((np.inf, np.nan, -np.inf)):
        if rows > 6 + i:
            x[5 + i, r.integers(cols)] = bad
    if rows > 4:
        x[4] = (r.normal(size=cols) * 2.0 ** -130).astype(np.float32)
        x[2] = 0
    if rows > 10:
        x[8] = (r.normal(size=cols) * 2.0 ** -95).astype(np.float32)
        x[9] = np.float32(3e38) * r.choice([-1, 0.5, 1], size=cols)
        x[10] = np.float32(-0.0)
    return x


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,extra", [(1, 1, 0), (3, 31, 1), (5, 128, 0), (7, 129, 3), (33, 1000, 8), (6, 2560, 0), (300, 260, 1),
                                             (11, 512, 0), (11, 513, 0), (12, 2048, 0), (12, 2049, 3), (12, 8192, 0), (13, 8193, 0),
                                             (12, 16384, 0), (3, 16385, 1), (4, 40000, 0), (3, 65536, 0)])
def test_quantize(type, rows, cols, extra):
    say("quantize", type, rows, cols, extra)
    x, values = hip.rows(special(rows, cols, rows + cols), type, extra)
    m, codes, scales = matrix(rows, cols)
    moe.i8_quantize_async(TYPES[type], x.ptr, m, stride=cols + extra)
    want, s = ref.i8_quantize(values)
    got, gs = codes.get(), scales.get()
    assert np.array_equal(gs[:rows], s.astype(np.float32), equal_nan=True) and gs[rows] == 7.0
    assert np.array_equal(got[:rows], ref.i8_padded(want)) and (got[rows] == 0x5A).all()
    out, _ = hip.rows(np.full((rows, cols), 7.0), type, extra, 1, 7.0)
    moe.i8_dequantize_async(m, TYPES[type], out.ptr, stride=cols + extra)
    back = out.get()
    assert (decode(back[rows:], type) == 7.0).all() and (decode(back[:, cols:], type) == 7.0).all()
    with np.errstate(over="ignore", invalid="ignore"):
        value = (want * s[:, None]).astype(np.float32)  # (a code's 8 and a scale's 24 bits: rounded once)
        assert np.array_equal(decode(back[:rows, :cols], type), decode(encode(value, type), type), equal_nan=True)


def test_many_rows():
    """More rows than a launch has work-groups: 300,000 of 5 values (four a work-group), 70,000 of 2100."""
    for rows, cols in ((300000, 5), (70000, 2100)):
        say("many rows", rows, cols)
        x = np.random.default_rng(cols).normal(size=(rows, cols)).astype(np.float32)
        xb = hip.put(x)
        m, codes, scales = matrix(rows, cols)
        moe.i8_quantize_async(moe.QT_F32, xb.ptr, m)
        some = np.r_[0:300, rows // 2:rows // 2 + 300, rows - 300:rows]
        want, s = ref.i8_quantize(x[some])
        assert np.array_equal(codes.get()[some], ref.i8_padded(want)) and np.array_equal(scales.get()[some], s.astype(np.float32))
        out = hip.full((rows, cols), 0)
        moe.i8_dequantize_async(m, moe.QT_F32, out.ptr)
        assert np.array_equal(out.get()[some], (want * s[:, None]).astype(np.float32))


def operand(rows, cols, seed, least=-127):
    r = np.random.default_rng(seed)
    return r.integers(least, 128, size=(rows, cols)), np.exp2(r.uniform(-12, 2, size=rows)).astype(np.float32).astype(np.float64)


def product(x, w, out="f32", extra=0, work_value=0xA5):
    """y of (codes, scales) pairs through i8_matmul_async, guards checked."""
    (xc, xs), (wc, ws) = x, w
    M, N, K = len(xc), len(wc), wc.shape[1]
    xm, *keep = matrix(M, K, xc, xs)
    wm, *keep2 = matrix(N, K, wc, ws)
    y, _ = hip.rows(np.full((M, N), 7.0), out, extra, 1, 7.0)
    n = moe.i8_matmul_work_bytes(wm, M)
    work = hip.full(n + 64, work_value, np.uint8)
    moe.i8_matmul_async(xm, wm, TYPES[out], y.ptr, work.ptr, n, y_stride=N + extra)
    got = decode(y.get(), out)
    assert (got[M:] == 7.0).all() and (got[:, N:] == 7.0).all() and (work.get()[n:] == work_value).all()
    return got[:M, :N]


def check(got, x, w, out):
    y, off = ref.i8_product(*x, *w)
    off = off + ref.EPS[out] * (np.abs(y) + off) + TINY[out]
    with np.errstate(over="ignore"):
        most = {"f32": 3.4e38, "f16": 65504.0, "bf16": 3.3e38}[out]
    fits = np.abs(y) + off < most
    assert (np.abs(got - y) <= off)[fits].all(), float((np.abs(got - y) / off)[fits].max())


# Few rows, each tile size, split k, sizes on and off every border.
SHAPES = [(1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 100, 1000), (5, 33, 64), (16, 2048, 1024), (16, 600, 9000), (1, 9000, 300), (3, 50, 8192),
          (17, 64, 128), (17, 1, 1), (33, 65, 127), (64, 64, 1000), (100, 130, 8200), (65, 1000, 257), (301, 2565, 1000), (128, 128, 65536),
          (700, 2100, 384), (2000, 1950, 200), (1800, 1804, 513), (3330, 4100, 640), (4096, 3329, 130), (20, 40, 5000),
          (40, 20000, 100), (40, 20000, 300), (40, 20000, 500), (40, 20000, 700), (512, 8192, 200), (520, 8000, 900), (1500, 1500, 130),
          (2688, 2048, 260), (3500, 3500, 1100), (3500, 3499, 1300), (16, 4096, 8192), (9, 5000, 8190), (17, 1500, 4100), (60, 3, 20000),
          (40, 40000, 130), (33000, 20, 129), (17, 33000, 3200), (100, 30000, 200)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul(M, N, K):
    say("matmul", M, N, K)
    x, w = operand(M, K, M + K), operand(N, K, N + K, -128)
    for out, extra in (("f32", 0), ("bf16", 3), ("f16", 8)):
        check(product(x, w, out, extra), x, w, out)


def test_largest_sums():
    """65536 products of -128 by -128: 2^30, the most that a sum holds."""
    say("largest sums")
    for M in (1, 40):
        x, w = (np.full((M, 65536), -128), np.ones(M)), (np.full((70, 65536), -128), np.ones(70))
        assert (product(x, w) == 2.0 ** 30).all()


def test_scales_that_are_no_numbers():
    """A row of x or of w with a scale of NaN makes its row or column of y NaN and nothing else."""
    say("nan scales")
    for M in (3, 40):
        x, w = operand(M, 200, 1), operand(50, 200, 2)
        clean = product(x, w)
        x[1][1], w[1][7] = np.nan, np.nan
        got = product(x, w)
        bad = np.zeros((M, 50), bool)
        bad[1], bad[:, 7] = True, True
        assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("M", [17, 64])
def test_whatever_the_work_buffer_held(M):
    say("work buffer", M)
    x, w = operand(M, 8200, 1), operand(130, 8200, 2)
    assert moe.i8_matmul_work_bytes(moe.I8Matrix(None, None, 130, 8200), M) > 0
    got = [product(x, w, work_value=v) for v in (0, 0xFF, 0x7F)]
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K,extra", [(1, 40, 2048, 0), (1, 9, 16384, 0), (4, 700, 4096, 1), (16, 48, 1024, 0), (16, 48, 1025, 3), (3, 33, 5, 2),
                                         (16, 16, 60000, 0), (17, 50, 300, 0), (150, 260, 1000, 5), (2, 8200, 2048, 0)])
def test_linear(type, M, N, K, extra):
    """The bits of the quantisation and the product one after the other, from the same floats, with rows of infinities and NaNs."""
    say("linear", type, M, N, K, extra)
    xf = special(M, K, M + K)
    xb, values = hip.rows(xf, type, extra)
    w = operand(N, K, 3)
    wm, *keep = matrix(N, K, *w)
    xm, *keep2 = matrix(M, K)
    moe.i8_quantize_async(TYPES[type], xb.ptr, xm, stride=K + extra)
    n = moe.i8_matmul_work_bytes(wm, M)
    work, y = room(n + 16), hip.full((M, N), 7.0)
    moe.i8_matmul_async(xm, wm, moe.QT_F32, y.ptr, work.ptr, n)
    want = y.get()
    n = moe.i8_linear_work_bytes(wm, M)
    work = room(n + 64)
    got, _ = hip.rows(np.full((M, N), 7.0), "f32", 2, 1, 7.0)
    moe.i8_linear_async(TYPES[type], xb.ptr, M, wm, moe.QT_F32, got.ptr, work.ptr, n, x_stride=K + extra, y_stride=N + 2)
    g = got.get()
    assert np.array_equal(g[:M, :N], want, equal_nan=True) and (g[M:] == 7.0).all() and (g[:, N:] == 7.0).all()
    assert (work.get()[n:] == 0xA5).all()
    x = ref.i8_quantize(values)
    fine = np.isfinite(x[1])
    check(want[fine], (x[0][fine], x[1][fine]), w, "f32")
    assert np.isnan(want[~fine]).all()


def test_far_rows():
    """w past 2^32 bytes and y past 2^32 elements' bytes: their last rows and columns."""
    say("far rows")
    N, K = 70000, 65536  # 4.6 GB of codes
    few = operand(64, K, 1)
    codes, scales = Raw(hip, N * K), hip.full(N, 1.0)
    codes.put(few[0].astype(np.int8), (N - 64) * K)
    w = moe.I8Matrix(codes.ptr, scales.ptr, N, K)
    for M in (2, 20):
        x = operand(M, K, 2)
        xm, *keep = matrix(M, K, *x)
        y = hip.full((M, N), 7.0)
        n = moe.i8_matmul_work_bytes(w, M)
        work = room(n + 16)
        moe.i8_matmul_async(xm, w, moe.QT_F32, y.ptr, work.ptr, n)
        got = y.get()
        check(got[:, -64:], x, (few[0], np.ones(64)), "f32")
        assert not got[:, :-64].any()


def test_graph_and_threads():
    """Linear products captured and replayed on new rows between eager calls; from four threads at once."""
    say("graph")
    N, K = 300, 640
    w = operand(N, K, 3)
    wm, *keep = matrix(N, K, *w)
    r = np.random.default_rng(1)
    for M in (4, 40):
        n = moe.i8_linear_work_bytes(wm, M)
        x = hip.full((M, K), 0)
        (wa, ya), (wb, yb) = ((room(n + 16), hip.full((M, N), 0)) for _ in range(2))
        s1, s2 = hip.stream(), hip.stream()
        launch = hip.capture(s1, lambda: moe.i8_linear_async(moe.QT_F32, x.ptr, M, wm, moe.QT_F32, ya.ptr, wa.ptr, n, stream=s1))
        for i in range(4):
            x.put(r.normal(size=(M, K)).astype(np.float32))
            launch()
            moe.i8_linear_async(moe.QT_F32, x.ptr, M, wm, moe.QT_F32, yb.ptr, wb.ptr, n, stream=s2)
            assert np.array_equal(ya.get(), yb.get())
            check(yb.get().astype(np.float64), ref.i8_quantize(x.get()), w, "f32")
    jobs = []
    for i, M in enumerate((1, 16, 50, 200)):
        x = hip.put(r.normal(size=(M, K)).astype(np.float32))
        n = moe.i8_linear_work_bytes(wm, M)
        jobs.append((M, x, room(n + 16), n, hip.full((M, N), 0), hip.stream()))

    def call(M, x, work, n, y, s):
        for _ in range(20):
            moe.i8_linear_async(moe.QT_F32, x.ptr, M, wm, moe.QT_F32, y.ptr, work.ptr, n, stream=s)

    threads = [threading.Thread(target=call, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for M, x, _, _, y, _ in jobs:
        check(y.get().astype(np.float64), ref.i8_quantize(x.get()), w, "f32")


def test_a_device_that_is_not_there():
    say("device")
    m, *keep = matrix(4, 128, *operand(4, 128, 1))
    y = hip.full((4, 4), 0)
    with pytest.raises(moe.MoeError) as e:
        moe.i8_matmul_async(m, m, moe.QT_F32, y.ptr, device=99)
    assert e.value.status == MOE_ERROR
    moe.i8_matmul_async(m, m, moe.QT_F32, y.ptr)
    assert y.get().all()
