"""Products of 8-bit integers and their experts on the GPU where addresses are far: results, weights and rows past 2^32 bytes in each
form of the kernels, and the experts' longest rows. Bounds as in tests/test_gpu_i8.py and tests/test_gpu_i8_experts.py."""
import numpy as np
import pytest

from tests import more_ref as ref
from tests.harness import moe
from tests.ops_dev import Raw, decode, encode, hip
from tests.test_gpu_i8 import check, matrix, operand, room, say
from tests.test_gpu_i8_experts import Model, check as check_experts, tokens

pytestmark = pytest.mark.gpu

FAR = 5 << 30  # bytes


# Few rows with four waves and with sixteen, quantised and floats; tiles of 64 in parts of k, of 64 with four buffers and with two, of
# 128 with four and with two, of 256.
@pytest.mark.parametrize("M,N,K,linear", [(3, 100, 300, False), (3, 40, 9000, False), (4, 100, 300, True), (16, 40, 1024, True),
                                          (17, 100, 3000, False), (512, 500, 200, False), (1500, 1500, 130, False), (17, 33000, 3200, False),
                                          (512, 8192, 200, False), (700, 8192, 200, False), (3500, 3500, 300, False)])
def test_far_results(M, N, K, linear):
    """y's rows so far apart that the last lie past 2^32 bytes; what is between them stays."""
    say("far results", M, N, K, linear)
    stride = FAR // 2 // M
    w = operand(N, K, N + K)
    wm, *keep = matrix(N, K, *w)
    y = Raw(hip, FAR, 0x5A)
    if linear:
        xf = np.random.default_rng(M).normal(size=(M, K)).astype(np.float32)
        x = ref.i8_quantize(xf)
        xb, n = hip.put(xf), moe.i8_linear_work_bytes(wm, M)
        work = room(n + 16)
        moe.i8_linear_async(moe.QT_F32, xb.ptr, M, wm, moe.QT_BF16, y.ptr, work.ptr, n, y_stride=stride)
    else:
        x = operand(M, K, M + K)
        xm, *keep2 = matrix(M, K, *x)
        n = moe.i8_matmul_work_bytes(wm, M)
        work = room(n + 16)
        moe.i8_matmul_async(xm, wm, moe.QT_BF16, y.ptr, work.ptr, n, y_stride=stride)
    some = np.unique(np.r_[np.linspace(0, M - 1, 60).astype(int), max(M - 20, 0):M])
    rows = [y.get(int(i) * stride * 2, ((N + 8) * 2,)).view(np.uint16) for i in some]
    assert all((r[N:] == 0x5A5A).all() for r in rows)
    check(np.stack([decode(r[:N], "bf16") for r in rows]), (x[0][some], x[1][some]), w, "bf16")


# Tiles of 64 with two buffers and with four, of 128, of 256 (few rows and 64 in parts do not reach so far, or are tested elsewhere).
@pytest.mark.parametrize("M,N,K", [(40, 1500000, 2944), (40, 70000, 65536), (200, 70000, 65536), (2000, 70000, 65536)])
def test_far_weights(M, N, K):
    """w's codes past 2^32 bytes: the last rows have values, the others are zeros."""
    say("far weights", M, N, K)
    few, last = 20, 64
    x, wl = operand(few, K, 1), operand(last, K, 2)
    at = np.arange(M) % few  # x's rows are these, over and over
    xm, *keep = matrix(M, K, x[0].astype(np.int8)[at], x[1][at])
    codes, scales = Raw(hip, N * K), hip.full(N, 1.0)
    assert N * K > 1 << 32
    codes.put(wl[0].astype(np.int8).view(np.uint8), (N - last) * K)
    scales.put(wl[1].astype(np.float32), (N - last) * 4)
    w = moe.I8Matrix(codes.ptr, scales.ptr, N, K)
    n = moe.i8_matmul_work_bytes(w, M)
    work, y = room(n + 16), Raw(hip, M * N * 2, 0x5A)
    moe.i8_matmul_async(xm, w, moe.QT_BF16, y.ptr, work.ptr, n)
    got = decode(y.get().view(np.uint16).reshape(M, N)[:, -last - 100:], "bf16")
    assert not got[:, :100].any()
    check(got[:, 100:], (x[0][at], x[1][at]), wl, "bf16")


@pytest.mark.parametrize("N", [20, 200])
def test_far_rows_of_x(N):
    """70000 rows of 65536 bf16 values, quantised to 4.6 GB of codes and multiplied: all zeros but the last."""
    say("far x", N)
    M, K, last = 70000, 65536, 40
    xf = np.random.default_rng(1).normal(size=(last, K)).astype(np.float32)
    raw = encode(xf, "bf16")
    x = Raw(hip, M * K * 2)
    x.put(raw.view(np.uint8), (M - last) * K * 2)
    w = operand(N, K, 2)
    wm, *keep = matrix(N, K, *w)
    n = moe.i8_linear_work_bytes(wm, M)
    work, y = Raw(hip, n + 64, 0xA5), hip.full((M, N), 7.0)
    moe.i8_linear_async(moe.QT_BF16, x.ptr, M, wm, moe.QT_F32, y.ptr, work.ptr, n)
    got = y.get()
    assert not got[:-last].any() and (work.get(n, (64,)) == 0xA5).all()
    check(got[-last:], ref.i8_quantize(decode(raw, "bf16")), w, "f32")


def test_experts_of_the_longest_rows():
    """The most tokens and ranks of the longest rows: 17 GB of fp32 values, so that down takes 256 columns at a time, 64 times over; x's
    rows over and over the same 60."""
    say("longest rows")
    T, H, F, E, K = 16384, 16384, 8, 3, 16
    model = Model(E, H, F, 6)
    x, ids, w = tokens(60, H, E, K, 9, 0.6, True)
    at = np.arange(T) % 60
    check_experts(model, x[at], ids[at], w[at], rows=np.r_[0:6, T // 2:T // 2 + 6, T - 6:T])


@pytest.mark.parametrize("T,H,F,E,K", [(1, 256, 64, 1, 16), (4, 300, 70, 2, 16), (10, 256, 64, 3, 16), (50, 256, 64, 2, 16)])
def test_more_ranks_than_experts(T, H, F, E, K):
    """A token names an expert several times: each time counts, in rank order."""
    say("ranks", T, H, F, E, K)
    check_experts(Model(E, H, F, T), *tokens(T, H, E, K, T, 0.2, True))
