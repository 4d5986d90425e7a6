"""The sums and roundings of the way back from the experts on the GPU, as the header states them, and rows for which one launch has
not enough threads.

Bounds. dw is a row's products in fp32: a lane has every 64th piece of kN neighbours (16 bytes; one element where a row is shorter),
its fused products added one chain to each place in a piece, then log2(kN) and six additions join them. Every operation is off by at
most 2^-24 of the sum of the products' sizes (2^-150 where it is denormal), so that dw is off by at most
(ceil(pieces / 64) + log2(kN) + 6) 2^-24 of it; 2^-11 of that covers the sizes' own growth by the roundings (at most 4104, for the
longest row, one on the other)."""
import numpy as np
import pytest

from tests import more_ref as ref
from tests.harness import moe
from tests.ops_dev import TYPES, Raw, decode, encode, hip
from tests.test_gpu_dispatch import say

pytestmark = pytest.mark.gpu

SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def steps(H, type):
    """How many roundings of the whole sum's size dw has at most."""
    n = 16 // SIZE[type]
    n = n if H >= n else 1
    pieces = -(-H // n)
    return -(-pieces // 64) + int(np.log2(n)) + 6


def gradient(dy, o, places, type, extra=0):
    """dw (T, K) of rows dy (T, H) and o (T K, H)."""
    (T, H), K = dy.shape, places.shape[1]
    dyb, dyv = hip.rows(dy, type, extra)
    ob, ov = hip.rows(o, type, extra)
    pb, dw = hip.put(places.astype(np.int32)), hip.full((T, K), 7.0)
    moe.Dispatch(8, K, H, TYPES[type]).combine_backward_async(dyb.ptr, T, pb.ptr, ob.ptr, None, dw.ptr, dy_stride=H + extra,
                                                               o_stride=H + extra)
    return dw.get(), dyv, ov


# A row shorter than a piece; of one piece and one more value; of 64 pieces, one less and one more; of some hundreds a lane.
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H", [1, 3, 7, 8, 9, 255, 256, 257, 511, 512, 513, 1001, 2048, 9000, 70001])
def test_weights_gradient(H, type):
    say("dw", H, type)
    T, K = 9, 3
    r = np.random.default_rng(H)
    places = r.permutation(T * K).reshape(T, K)
    for positive in (False, True):
        dy, o = r.normal(size=(T, H)), r.normal(size=(T * K, H))
        if positive:  # (the sum is its sizes' sum: the bound is what the roundings reach, not the terms' cancellation)
            dy, o = np.abs(dy), np.abs(o)
        got, dyv, ov = gradient(dy, o, places, type, 3)
        terms = dyv[:, None, :] * ov[places]
        off = steps(H, type) * 2.0 ** -24 * (1 + 2.0 ** -11) * np.abs(terms).sum(-1) + H * 2.0 ** -149
        assert (np.abs(got - terms.sum(-1)) <= off).all(), float((np.abs(got - terms.sum(-1)) / off).max())


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("H", [5, 260, 4097])
def test_weights_gradient_whatever_the_others(H, type):
    """The order of a row's sum goes by n_embd and type alone: one token's dw has the same bits by itself and in any batch."""
    say("dw alone", H, type)
    r = np.random.default_rng(H)
    dy, o = r.normal(size=(1, H)), r.normal(size=(1, H))
    alone = gradient(dy, o, np.zeros((1, 1), int), type)[0][0, 0]
    for T, K, t, k, extra in ((1, 16, 0, 11, 0), (7, 3, 5, 0, 1), (300, 10, 299, 9, 8)):
        places = r.permutation(T * K).reshape(T, K)
        dys, os = r.normal(size=(T, H)), r.normal(size=(T * K, H))
        dys[t], os[places[t, k]] = dy[0], o[0]
        assert gradient(dys, os, places, type, extra)[0][t, k] == alone


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_roundings_of_the_rows_gradient(type):
    """dout is the product in fp32 rounded to the type, bit for bit, also where that is not the nearest of the exact product."""
    say("dout", type)
    T, K, H = 300, 4, 1001
    r = np.random.default_rng(5)
    places = r.permutation(T * K).reshape(T, K)
    dyb, dy = hip.rows(r.normal(size=(T, H)), type)
    w = r.normal(size=(T, K)).astype(np.float32)
    pb, wb, dout = hip.put(places.astype(np.int32)), hip.put(w), hip.put(encode(np.zeros((T * K, H)), type))
    moe.Dispatch(8, K, H, TYPES[type]).combine_backward_async(dyb.ptr, T, pb.ptr, None, dout.ptr, None, wb.ptr)
    exact = dy[:, None, :] * w[:, :, None].astype(np.float64)  # (24 and at most 24 bits: whole in a double)
    want = np.empty((T * K, H), dout.dtype)
    want[places.ravel()] = encode(exact.astype(np.float32), type).reshape(T * K, H)
    assert np.array_equal(dout.get(), want)


def test_more_pieces_than_a_launch_has_threads():
    """17000 rows of 2^20 values (35.7 GB, 34.8 million runs of 64 pieces) there and back: two launches each, of 16384 tokens and the
    rest, and both gradients."""
    say("many pieces")
    T, H = 17000, 1 << 20
    d = moe.Dispatch(3, 1, H)
    ids = np.random.default_rng(3).integers(0, 3, size=(T, 1)).astype(np.int32)
    ids[7] = -1
    order, places, offsets = ref.dispatch(ids, 3)
    some = np.r_[0, 1, 7, 8000, 16383, 16384, 16385, T - 1]  # tokens with rows of their own; the others' are ones
    r = np.random.default_rng(4)
    rows = encode(r.integers(-100, 100, size=(len(some), H)), "bf16")
    x, xs = Raw(hip, T * H * 2, 0x3F), Raw(hip, T * H * 2, 0x11)  # (0x3f3f: 191 / 256)
    for t, row in zip(some, rows):
        x.put(row.view(np.uint8), int(t) * H * 2)
    idb, pb = hip.put(ids), hip.full((T, 1), 0, np.int32)
    ob, fb = hip.full(T, 0, np.int32), hip.full(4, 0, np.int32)
    work = hip.full(d.work_bytes(T) + 16, 0, np.uint8)
    say("dispatch")
    d.dispatch_async(x.ptr, T, idb.ptr, xs.ptr, ob.ptr, pb.ptr, fb.ptr, work.ptr, work.nbytes)
    assert np.array_equal(ob.get(), order) and np.array_equal(pb.get(), places) and np.array_equal(fb.get(), offsets)

    def row(buf, i):
        return buf.get(int(i) * H * 2, (H * 2,)).view(np.uint16)

    for t, want in zip(some, rows):
        if places[t, 0] >= 0:
            assert np.array_equal(row(xs, places[t, 0]), want), t
    assert (row(xs, places[16386, 0]) == 0x3F3F).all() and (row(xs, T - 1) == 0x1111).all()  # (no assignment is last)
    y = Raw(hip, T * H * 2, 0x55)
    w = hip.put(np.full((T, 1), 2.0, np.float32))
    say("combine")
    d.combine_async(xs.ptr, T, pb.ptr, y.ptr, w.ptr)
    for t, want in zip(some, rows):
        got = decode(row(y, t), "bf16")
        assert np.array_equal(got, np.zeros(H) if t == 7 else 2 * decode(want, "bf16")), t
    assert (decode(row(y, 16386), "bf16") == 2 * 191 / 256).all()
    dw = hip.full((T, 1), 7.0)
    say("combine backward")
    d.combine_backward_async(x.ptr, T, pb.ptr, xs.ptr, y.ptr, dw.ptr, w.ptr)
    got = dw.get()
    for t, want in zip(some, rows):
        sum_of = (decode(want, "bf16") ** 2).sum()
        assert got[t, 0] == 0.0 if t == 7 else abs(got[t, 0] - sum_of) <= steps(H, "bf16") * 2.0 ** -24 * (1 + 2.0 ** -11) * sum_of
        if t != 7:
            assert np.array_equal(decode(row(y, places[t, 0]), "bf16"), 2 * decode(want, "bf16"))
    say("dispatch backward")
    d.dispatch_backward_async(xs.ptr, T, pb.ptr, y.ptr)
    for t, want in zip(some, rows):
        assert np.array_equal(decode(row(y, t), "bf16"), np.zeros(H) if t == 7 else decode(want, "bf16"))
