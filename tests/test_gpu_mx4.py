"""Microscaled 4-bit floats on the GPU: quantisation and its inverse byte for byte, the products against sums in 64 bits.

A product's bound: the values' products are exact, at most K / 32 + 24 additions in fp32 round them (a matrix instruction
adds 32 to 128 of them, splits of k are joined), each by at most 2^-24 of the terms' absolute sum S, twice that allowed;
then one rounding to the result's type."""
import numpy as np
import pytest

from tests import ops_ref as ref
from tests.harness import moe
from tests.ops_dev import TYPES, Raw, decode, encode, hip

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def room(*shape):
    return hip.full(shape, 0xA5, np.uint8)


def matrix(rows, cols, codes=None, scales=None):
    """An Mx4Matrix with a guard row behind it, and its buffers."""
    c = ref.pad128(cols)
    bc, bs = room(rows + 1, c // 2), room(rows * c // 32 + 64)
    if codes is not None:
        bc.put(codes)
        bs.put(scales.ravel())
    return moe.Mx4Matrix(bc.ptr, bs.ptr, rows, cols), bc, bs


def special(rows, cols, seed):
    """Normal rows of different sizes, with zeros, halves between codes, subnormals, powers of two, infinities, NaNs."""
    r = np.random.default_rng(seed)
    x = (r.normal(size=(rows, cols)) * np.exp2(r.integers(-20, 20, size=(rows, 1)))).astype(np.float32)
    kinds = [np.float32(0), np.float32(-0.0), np.float32(np.inf), np.float32(np.nan), np.float32(-np.inf)]
    for i in range(0, rows, 3):
        x[i] = np.float32(2.0 ** float(r.integers(-8, 8))) * r.choice(np.concatenate([ref.BORDERS, ref.VALUES]), size=cols)
    for i in range(1, rows, 5):
        x[i, r.integers(cols)] = kinds[i % len(kinds)]
    if rows > 4:
        x[4] = (r.normal(size=cols) * 2.0 ** -130).astype(np.float32)
        x[2] = 0
    return x


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,extra", [(1, 1, 0), (3, 31, 1), (5, 32, 0), (2, 33, 7), (7, 128, 0), (11, 129, 3),
                                             (33, 1000, 8), (6, 2560, 0), (300, 260, 1)])
def test_quantize(type, rows, cols, extra):
    say("quantize", type, rows, cols, extra)
    x, values = hip.rows(special(rows, cols, rows + cols), type, extra)
    m, codes, scales = matrix(rows, cols)
    moe.mx4_quantize_async(TYPES[type], x.ptr, m, stride=cols + extra)
    want_c, want_s = ref.mx4_quantize(values)
    n = want_s.size
    got_c, got_s = codes.get(), scales.get()
    assert np.array_equal(got_s[:n], want_s.ravel())
    assert np.array_equal(got_c[:rows], want_c)
    assert (got_s[n:] == 0xA5).all() and (got_c[rows:] == 0xA5).all()


def test_quantize_every_scale():
    """Blocks of every size from the smallest subnormal to the largest float, with values on and beside the borders."""
    say("every scale")
    rows = []
    for e in range(-149, 128):
        top = np.float64(2.0) ** e
        rows.append(np.concatenate([top * np.array([1, 1.25, 1.75, 0.99999994, 1.9999999]),
                                    top / 4 * ref.BORDERS, top / 4 * ref.BORDERS * (1 + 2.0 ** -20),
                                    top / 4 * ref.BORDERS * (1 - 2.0 ** -20), -top / 4 * ref.VALUES[:6]]))
    x = np.clip(np.array(rows), -3.4028234663852886e38, 3.4028234663852886e38).astype(np.float32)
    b, values = hip.rows(x, "f32")
    m, codes, scales = matrix(*x.shape)
    moe.mx4_quantize_async(moe.QT_F32, b.ptr, m)
    want_c, want_s = ref.mx4_quantize(values)
    assert np.array_equal(scales.get()[:want_s.size], want_s.ravel())
    assert np.array_equal(codes.get()[:len(x)], want_c)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols,extra", [(128, 0), (97, 2)])
def test_dequantize_every_value(type, cols, extra):
    """Every code under every scale byte, rounded once to the type."""
    say("dequantize", type, cols)
    r = np.random.default_rng(1)
    codes = r.integers(0, 256, size=(256, 64)).astype(np.uint8)
    codes[:, :16] = np.arange(0, 256, 17)[None]  # each code, twice in a byte
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 4, 1)
    m, c, s = matrix(256, cols, codes, scales)
    out, _ = hip.rows(np.full((256, cols), 7.0), type, extra, fill=7.0)
    moe.mx4_dequantize_async(m, TYPES[type], out.ptr, stride=cols + extra)
    with np.errstate(over="ignore"):
        want = decode(encode(ref.mx4_values(codes, scales, cols).astype(np.float32), type), type)
    got = decode(out.get(), type)
    assert np.array_equal(got[:, :cols], want, equal_nan=True)
    assert (got[:, cols:] == 7.0).all()


def random_mx4(rows, cols, seed, spread=3):
    """A matrix of random codes, its scales within spread of a half: the description, its buffers, the values in 64 bits."""
    r = np.random.default_rng(seed)
    c = ref.pad128(cols)
    codes = r.integers(0, 256, size=(rows, c // 2)).astype(np.uint8)
    scales = r.integers(126 - spread, 127 + spread, size=(rows, c // 32)).astype(np.uint8)
    keep = np.arange(c) < cols  # codes past cols are 0
    codes &= (keep[0::2] * 15 | keep[1::2] * 240).astype(np.uint8)
    m, bc, bs = matrix(rows, cols, codes, scales)
    return m, (bc, bs), ref.mx4_values(codes, scales, cols), codes, scales


def close(got, x, w, type):
    y, S = x @ w.T, np.abs(x) @ np.abs(w).T
    bound = 2 * (x.shape[1] / 32 + 24) * 2.0 ** -24 * S
    bound = bound + ref.EPS[type] * (np.abs(y) + bound)
    assert np.all(np.abs(got - y) <= bound), float((np.abs(got - y) - bound).max())


SHAPES = [(1, 1, 1), (1, 16, 128), (2, 65, 640), (5, 300, 2048), (1, 2049, 1000), (16, 129, 4000), (17, 33, 129),
          (33, 512, 256), (64, 100, 1000), (65, 257, 384), (130, 70, 4096), (256, 256, 512), (301, 515, 1000), (513, 300, 640),
          (17, 40, 8192), (48, 70, 16000), (20, 33, 5000), (1, 8200, 1920), (15, 100, 1024), (1800, 2000, 300), (1750, 2001, 640)]


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul(M, N, K, out):
    say("matmul", M, N, K, out)
    x, xb, xv, _, _ = random_mx4(M, K, M + K, 1)
    w, wb, wv, _, _ = random_mx4(N, K, N + K + 1, 1)
    extra = (M + N) % 4
    y, _ = hip.rows(np.full((M, N), 7.0), out, extra, 1, 7.0)
    n = moe.mx4_matmul_work_bytes(w, M)
    work = room(n + 64)
    moe.mx4_matmul_async(x, w, TYPES[out], y.ptr, work.ptr, n, y_stride=N + extra)
    got = decode(y.get(), out)
    close(got[:M, :N], xv, wv, out)
    assert (got[M:] == 7.0).all() and (got[:, N:] == 7.0).all() and (work.get()[n:] == 0xA5).all()


@pytest.mark.parametrize("M,N,K", [(3700, 3601, 130), (3601, 3700, 700), (4000, 3600, 900)])
def test_matmul_of_the_largest_tiles(M, N, K):
    """Some rows and columns of y against sums in 64 bits, the others by their checksums along both axes: x times w's columns'
    sum, and x's rows' sum times w."""
    say("large tiles", M, N, K)
    x, xb, xv, _, _ = random_mx4(M, K, M + K, 1)
    w, wb, wv, _, _ = random_mx4(N, K, N + K + 1, 1)
    y = hip.full((M + 1, N), 7)
    n = moe.mx4_matmul_work_bytes(w, M)
    work = room(n + 64)
    moe.mx4_matmul_async(x, w, moe.QT_F32, y.ptr, work.ptr, n)
    got = y.get().astype(np.float64)
    assert (got[M:] == 7.0).all()
    got = got[:M]
    rows = np.r_[0:3, 200:320:7, M - 70:M]
    close(got[rows], xv[rows], wv, "f32")
    close(got[:, N - 70:], xv, wv[N - 70:], "f32")
    # A sum of n results is off by their bounds' sum: the same bound, on the absolute values' sum.
    for v, want, S in ((got.sum(0), xv.sum(0) @ wv.T, np.abs(xv).sum(0) @ np.abs(wv).T),
                       (got.sum(1), xv @ wv.sum(0), np.abs(xv) @ np.abs(wv).sum(0))):
        assert np.all(np.abs(v - want) <= (2 * (K / 32 + 24) + 2) * 2.0 ** -24 * S)


@pytest.mark.parametrize("type,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(M, N, K, type, out):
    say("linear", M, N, K, type, out)
    r = np.random.default_rng(M * N + K)
    extra = (M + N) % 4
    x, values = hip.rows(r.normal(size=(M, K)), type, extra)
    w, wb, wv, _, _ = random_mx4(N, K, N, 1)
    y, _ = hip.rows(np.full((M, N), 7.0), out, extra, 1, 7.0)
    n = moe.mx4_linear_work_bytes(w, M)
    work = room(n + 64)
    moe.mx4_linear_async(TYPES[type], x.ptr, M, w, TYPES[out], y.ptr, work.ptr, n, x_stride=K + extra, y_stride=N + extra)
    got = decode(y.get(), out)
    close(got[:M, :N], ref.mx4(values), wv, out)
    assert (got[M:] == 7.0).all() and (got[:, N:] == 7.0).all() and (work.get()[n:] == 0xA5).all()


@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_nans_stay_in_their_rows(M):
    """A row of x with a NaN or an infinity, a row of w with a NaN block: only y's row and column are NaN."""
    say("nan rows", M)
    N, K = 200, 700
    x = np.random.default_rng(M).normal(size=(M, K)).astype(np.float32)
    x[M // 2, 650] = np.inf if M % 2 else np.nan
    b, _ = hip.rows(x, "f32")
    w, wb, _, _, scales = random_mx4(N, K, 5, 1)
    scales[37, 3] = 255
    wb[1].put(scales.ravel())
    y = hip.full((M, N), 0)
    work = room(moe.mx4_linear_work_bytes(w, M) + 16)
    moe.mx4_linear_async(moe.QT_F32, b.ptr, M, w, moe.QT_F32, y.ptr, work.ptr, work.nbytes)
    nan = np.isnan(y.get())
    assert nan[M // 2].all() and nan[:, 37].all()
    nan[M // 2], nan[:, 37] = False, False
    assert not nan.any()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_extreme_scales(M):
    """Rows whose scales are far from one: the sums stay within fp32's own range of them."""
    say("extreme scales", M)
    N, K = 96, 512
    x, xb, _, codes, scales = random_mx4(M, K, 3, 0)
    w, wb, _, wcodes, wscales = random_mx4(N, K, 4, 0)
    scales[:] = 17
    wscales[:] = np.where(np.arange(N)[:, None] % 2, 230, 60)
    xb[1].put(scales.ravel())
    wb[1].put(wscales.ravel())
    y = hip.full((M, N), 0)
    work = room(moe.mx4_matmul_work_bytes(w, M) + 16)
    moe.mx4_matmul_async(x, w, moe.QT_F32, y.ptr, work.ptr, work.nbytes)
    xv, wv = ref.mx4_values(codes, scales, K), ref.mx4_values(wcodes, wscales, K)
    got, want, S = y.get().astype(np.float64), xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    # (products below 2^-126 may be flushed: K of them)
    assert np.all(np.abs(got - want) <= 2 * (K / 32 + 24) * 2.0 ** -24 * S + 2.0 ** -24 * np.abs(want) + K * 2.0 ** -126)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_graph_and_streams(M):
    """Captured on a stream of its own, replayed between other work on new inputs: each replay is the eager result."""
    say("graph", M)
    N, K = 300, 640
    r = np.random.default_rng(M)
    w, wb, wv, _, _ = random_mx4(N, K, 9, 1)
    x, y, z = hip.full((M, K), 0), hip.full((M, N), 0), hip.full((M, N), 0)
    work, work2 = (room(moe.mx4_linear_work_bytes(w, M) + 16) for _ in range(2))
    s, q = hip.stream(), hip.stream()

    def call(out, wk, stream):
        moe.mx4_linear_async(moe.QT_F32, x.ptr, M, w, moe.QT_F32, out.ptr, wk.ptr, wk.nbytes, stream=stream)

    launch = hip.capture(s, lambda: call(y, work, s))
    for i in range(4):
        x.put(r.normal(size=(M, K)))
        y.put(np.full((M, N), 7.0))
        launch()
        call(z, work2, q)
        a, b = y.get(), z.get()
        assert np.array_equal(a, b)
        close(b.astype(np.float64), ref.mx4(x.get()), wv, "f32")


def test_far_offsets():
    """Rows past 2^32 elements and past 2^32 bytes of codes."""
    say("far offsets")
    rows, cols = (1 << 17) + 40, 1 << 16  # 2^33 elements: 17 GB of bf16, 4.3 GB of codes
    x = Raw(hip, rows * cols * 2)
    last = encode(np.random.default_rng(1).normal(size=(40, cols)), "bf16")
    x.put(last.view(np.uint8), (rows - 40) * cols * 2)
    codes, scales = Raw(hip, rows * cols // 2, 0xFF), Raw(hip, rows * cols // 32, 0xFF)
    m = moe.Mx4Matrix(codes.ptr, scales.ptr, rows, cols)
    moe.mx4_quantize_async(moe.QT_BF16, x.ptr, m)
    want_c, want_s = ref.mx4_quantize(decode(last, "bf16"))
    assert np.array_equal(codes.get((rows - 40) * cols // 2, (40, cols // 2)), want_c)
    assert np.array_equal(scales.get((rows - 40) * cols // 32, (40, cols // 32)), want_s)
    assert not codes.get((rows - 80) * cols // 2, (40, cols // 2)).any() and not codes.get(0, (40, cols // 2)).any()
    x.fill(0x11)
    moe.mx4_dequantize_async(m, moe.QT_BF16, x.ptr)
    got = decode(x.get((rows - 40) * cols * 2, (40, cols * 2)).view(np.uint16), "bf16")
    assert np.array_equal(got, ref.mx4_values(want_c, want_s, cols))
    x.free()
    # The matrix as a product's w: its last rows.
    v, vb, vv, _, _ = random_mx4(1, cols, 2, 0)
    y = hip.full((1, rows), 0)
    work = room(moe.mx4_matmul_work_bytes(m, 1) + 16)
    moe.mx4_matmul_async(v, m, moe.QT_F32, y.ptr, work.ptr, work.nbytes)
    close(y.get()[:, -40:].astype(np.float64), vv, ref.mx4_values(want_c, want_s, cols), "f32")


def test_no_such_device():
    """A device that is not there is an error of that call alone."""
    x = np.random.default_rng(2).normal(size=(3, 200)).astype(np.float32)
    b = hip.put(x)
    m, codes, scales = matrix(3, 200)
    for device in (99, -1):
        with pytest.raises(moe.MoeError):
            moe.mx4_quantize_async(moe.QT_F32, b.ptr, m, device=device)
        assert hip.rt.hipGetLastError() == 0  # nothing is left for whoever asks next
    assert (codes.get() == 0xA5).all()
    moe.mx4_quantize_async(moe.QT_F32, b.ptr, m)
    assert np.array_equal(codes.get()[:3], ref.mx4_quantize(x.astype(np.float64))[0])


def test_nothing_to_do():
    m, codes, scales = matrix(0, 64)
    moe.mx4_quantize_async(moe.QT_F32, codes.ptr, m)
    moe.mx4_dequantize_async(m, moe.QT_F32, codes.ptr)
    w, wb, _, _, _ = random_mx4(8, 64, 1)
    y = hip.full((1, 8), 7)
    moe.mx4_matmul_async(m, w, moe.QT_F32, y.ptr)
    moe.mx4_linear_async(moe.QT_F32, codes.ptr, 0, w, moe.QT_F32, y.ptr, None, 0)
    assert (y.get() == 7.0).all() and (codes.get() == 0xA5).all()


def test_most_rows():
    """As many rows as a matrix may have, of two steps each: more values than a launch has threads for, there and back."""
    say("most rows")
    rows, cols = 1 << 27, 129  # 35 GB of fp16, 17 GB of codes
    x = Raw(hip, rows * cols * 2)
    r = np.random.default_rng(3)
    at = (0, rows // 2 - 50, rows - 100)
    parts = [encode(r.normal(size=(100, cols)), "f16") for _ in at]
    for a, part in zip(at, parts):
        x.put(part.view(np.uint8), a * cols * 2)
    codes, scales = Raw(hip, rows * 128, 0xFF), Raw(hip, rows * 8, 0xFF)
    m = moe.Mx4Matrix(codes.ptr, scales.ptr, rows, cols)
    moe.mx4_quantize_async(moe.QT_F16, x.ptr, m)
    want = [ref.mx4_quantize(decode(p, "f16")) for p in parts]
    for a, (c, s) in zip(at, want):
        assert np.array_equal(codes.get(a * 128, (100, 128)), c) and np.array_equal(scales.get(a * 8, (100, 8)), s)
    assert not codes.get(100 * 128, (1 << 20,)).any() and not codes.get((rows - (1 << 13)) * 128 - 100 * 128, (1 << 20,)).any()
    x.fill(0x11)
    moe.mx4_dequantize_async(m, moe.QT_F16, x.ptr)
    for a, (c, s) in zip(at, want):
        assert np.array_equal(decode(x.get(a * cols * 2, (100, cols * 2)).view(np.float16), "f16"), ref.mx4_values(c, s, cols))
    assert not x.get(100 * cols * 2, (1 << 20,)).any()


@pytest.mark.parametrize("M,N,K", [(1, 64, 640), (40, 100, 8192), (300, 200, 700)])
def test_whatever_the_work_buffer_held(M, N, K):
    say("work buffer", M, N, K)
    x, _ = hip.rows(np.random.default_rng(M).normal(size=(M, K)), "f32")
    w, wb, _, _, _ = random_mx4(N, K, 9, 1)
    y = hip.full((M, N), 0)
    n = moe.mx4_linear_work_bytes(w, M)
    work = room(n)
    got = []
    for value in (0x00, 0xFF, 0x7F):
        work.put(np.full(n, value, np.uint8))
        moe.mx4_linear_async(moe.QT_F32, x.ptr, M, w, moe.QT_F32, y.ptr, work.ptr, n)
        got.append(y.get())
    assert np.isfinite(got[0]).all() and all(np.array_equal(got[0], g) for g in got[1:])
