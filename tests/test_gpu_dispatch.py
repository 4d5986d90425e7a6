"""Tokens sorted by expert and back on the GPU, and the gradients: orders and copied rows exactly, sums against 64 bits.

Bounds: a token's sum is K fused products in fp32, each off by at most 2^-24 of the terms' sizes' sum, and one rounding to the
type; a weight's gradient is n_embd fused products in 64 chains and six additions, each off by at most 2^-24 of the sizes' sum."""
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


def draw_ids(T, K, E, seed, dropped=0.1, skew=0.0):
    r = np.random.default_rng(seed)
    ids = r.integers(0, E, size=(T, K))
    ids = np.where(r.random((T, K)) < skew, E // 2, ids)
    ids = np.where(r.random((T, K)) < dropped, r.choice([-1, E, -(1 << 31), (1 << 31) - 1], size=(T, K)), ids)
    return ids.astype(np.int32)


class Call:
    """A dispatch's buffers, each with guards behind it, and its results checked against the plain form."""

    def __init__(self, ids, E, H, type="f32", extra=0, rows=True, seed=0, stream=None):
        T, K = ids.shape
        self.T, self.K, self.E, self.H, self.type, self.extra = T, K, E, H, type, extra
        self.d = moe.Dispatch(E, K, H, TYPES[type])
        self.ids = hip.put(np.concatenate([ids.ravel(), [3]]).astype(np.int32))
        self.order, self.places = hip.full(T * K + 1, 77, np.int32), hip.full(T * K + 1, 77, np.int32)
        self.offsets = hip.full(E + 2, 77, np.int32)
        self.n = self.d.work_bytes(T)
        self.work = hip.full(self.n + 64, 0xA5, np.uint8)
        if rows:
            x = np.random.default_rng(seed).normal(size=(T, H))
            self.x, _ = hip.rows(x, type, extra)
            self.xs, _ = hip.rows(np.full((T * K, H), 7.0), type, extra, 1, 7.0)
        self.rows = rows

    def run(self, stream=None):
        s = self.H + self.extra
        self.d.dispatch_async(self.x.ptr if self.rows else None, self.T, self.ids.ptr, self.xs.ptr if self.rows else None,
                              self.order.ptr, self.places.ptr, self.offsets.ptr, self.work.ptr, self.n, x_stride=s, xs_stride=s,
                              stream=stream)

    def check(self, ids):
        n = ids.size
        order, places, offsets = ref.dispatch(ids, self.E)
        got = [b.get() for b in (self.order, self.places, self.offsets)]
        assert [g[-1] for g in got] == [77] * 3 and (self.work.get()[self.n:] == 0xA5).all()
        assert np.array_equal(got[2][:-1], offsets)
        assert np.array_equal(got[0][:n], order) and np.array_equal(got[1][:n], places.ravel())
        if self.rows:
            x, xs = self.x.get(), self.xs.get()
            P = offsets[-1]
            assert np.array_equal(xs[:P, :self.H], x[order[:P] // self.K, :self.H])
            seven = encode(np.float32([7.0]), self.type)[0]
            assert (xs[P:] == seven).all() and (xs[:, self.H:] == seven).all()


# One token to several slices of ids; rows of one value, of fewer and of more than 32 pieces, of whole pieces and not.
@pytest.mark.parametrize("T,K,E,H", [(1, 1, 1, 1), (1, 10, 512, 2048), (3, 4, 7, 33), (8, 10, 512, 100), (16, 16, 64, 515),
                                     (64, 16, 8, 260), (65, 16, 8, 129), (200, 7, 2, 17), (255, 16, 512, 64), (300, 14, 100, 1000),
                                     (1025, 4, 511, 250), (2000, 10, 60, 40), (5000, 3, 512, 7), (17, 2, 5, 20000), (160, 16, 40, 2700), (161, 16, 40, 130), (2560, 1, 33, 9),
                                     (700, 3, 512, 5000), (2, 16, 20, 70001)])
def test_dispatch(T, K, E, H):
    for type, extra, dropped, skew in (("f32", 0, 0.0, 0.0), ("bf16", 3, 0.2, 0.7), ("f16", 0, 0.1, 0.0)):
        say("dispatch", T, K, E, H, type)
        ids = draw_ids(T, K, E, T + K, dropped, skew)
        c = Call(ids, E, H, type, extra)
        c.run()
        c.check(ids)


@pytest.mark.parametrize("T,K", [(5, 3), (70, 16), (150, 16), (400, 16)])
def test_edges_of_ids(T, K):
    """All on the first, on the last, on no expert; the same one in each rank; all in order and in reverse."""
    say("ids", T, K)
    E = 512
    n = np.arange(T * K).reshape(T, K)
    for ids in (np.zeros((T, K)), np.full((T, K), E - 1), np.full((T, K), -1), n // K % E, n * E // n.size, E - 1 - n * E // n.size):
        ids = ids.astype(np.int32)
        c = Call(ids, E, 48)
        c.run()
        c.check(ids)


@pytest.mark.parametrize("T", [4096 * 4 // 16, 1 << 16, (1 << 18) + 777, 1 << 20])
def test_many_ids(T):
    """One slice exactly; slices of the smallest size; longer ones, up to the most tokens. Only the order."""
    say("many ids", T)
    ids = draw_ids(T, 16, 500, 3, 0.05, 0.3)
    c = Call(ids, 500, 16, rows=False)
    c.run()
    c.check(ids)


def test_far_rows():
    """Sorted rows past 2^32 bytes: 32768 tokens of 16 ranks and 4200 values, 4.4 GB, and back."""
    T, K, E, H = 32768, 16, 64, 4200
    say("far rows")
    ids = draw_ids(T, K, E, 5, 0.0)
    order, places, _ = ref.dispatch(ids, E)
    r = np.random.default_rng(0)
    x = encode(r.integers(-128, 128, size=(T, H)), "bf16")
    d = moe.Dispatch(E, K, H)
    xb, idb = hip.put(x), hip.put(ids)
    xs = Raw(hip, T * K * H * 2)
    ob, pb, fb = hip.full(T * K, 0, np.int32), hip.full(T * K, 0, np.int32), hip.full(E + 1, 0, np.int32)
    work = hip.full(d.work_bytes(T) + 16, 0, np.uint8)
    d.dispatch_async(xb.ptr, T, idb.ptr, xs.ptr, ob.ptr, pb.ptr, fb.ptr, work.ptr, work.nbytes)
    assert np.array_equal(ob.get(), order)
    for p in (0, T * K // 2, T * K - 2000):
        got = xs.get(p * H * 2, (2000, H * 2)).view(np.uint16)
        assert np.array_equal(got, x[order[p:p + 2000] // K])
    y = hip.full((T, H), 0, np.uint16)
    d.combine_async(xs.ptr, T, pb.ptr, y.ptr)  # sixteen times a whole number of seven bits: exact
    assert np.array_equal(decode(y.get(), "bf16"), 16 * decode(x, "bf16"))
    dw = hip.full((T, K), 0)
    d.combine_backward_async(xb.ptr, T, pb.ptr, xs.ptr, None, dw.ptr)
    t = np.r_[0:50, T - 50:T]
    v = decode(x[t], "bf16")
    assert np.abs(dw.get()[t] - (v * v).sum(-1)[:, None]).max() <= (H / 64 + 16) * 2.0 ** -24 * (v * v).sum(-1).max()


def back(T, K, E, H, type, extra, seed, weighted=True):
    """places, o (NaN in the rows without an assignment), w (NaN where nothing is placed) and their buffers."""
    r = np.random.default_rng(seed)
    ids = draw_ids(T, K, E, seed, 0.2)
    ids[T // 2] = -1
    _, places, offsets = ref.dispatch(ids, E)
    o = r.normal(size=(T * K, H))
    o[offsets[-1]:] = np.nan
    ob, ov = hip.rows(o, type, extra, 1)
    w = np.where(places >= 0, r.normal(size=(T, K)), np.nan).astype(np.float32) if weighted else None
    return places, ov, w, hip.put(places.astype(np.int32)), ob, hip.put(w) if weighted else None


BACK = [(1, 1, 1, 1), (1, 10, 512, 2048), (8, 10, 64, 2048), (7, 16, 20, 515), (33, 9, 8, 129), (300, 4, 16, 1001), (100, 8, 40, 31),
        (2000, 5, 60, 6), (5, 3, 4, 9000)]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,K,E,H", BACK)
def test_combine(T, K, E, H, type):
    for extra, weighted in ((0, True), (5, False)):
        say("combine", T, K, E, H, type, extra, weighted)
        places, o, w, pb, ob, wb = back(T, K, E, H, type, extra, T + H, weighted)
        y, _ = hip.rows(np.full((T, H), 7.0), type, extra, 1, 7.0)
        d = moe.Dispatch(E, K, H, TYPES[type])
        d.combine_async(ob.ptr, T, pb.ptr, y.ptr, wb.ptr if weighted else None, o_stride=H + extra, y_stride=H + extra)
        got = decode(y.get(), type)
        assert (got[T:] == 7.0).all() and (got[:, H:] == 7.0).all()
        want, size = ref.combine(o, places, w)
        off = (K + 1) * 2.0 ** -24 * size
        off = off + ref.EPS[type] * (np.abs(want) + off) + TINY[type]
        assert (np.abs(got[:T, :H] - want) <= off).all()
        assert not got[T // 2, :H].any()
        if not weighted:  # the gradient of the dispatch is this sum
            again, _ = hip.rows(np.full((T, H), 7.0), type, extra, 1, 7.0)
            d.dispatch_backward_async(ob.ptr, T, pb.ptr, again.ptr, dxs_stride=H + extra, dx_stride=H + extra)
            assert np.array_equal(again.get(), y.get())


def test_combine_ignores_places_that_are_none():
    """A place past the rows, or negative, is not followed, and its weight not used; repeated places add each time."""
    say("places")
    T, K, H = 3, 4, 40
    o = np.random.default_rng(1).normal(size=(T * K, H)).astype(np.float32)
    places = np.array([[0, 12, -5, 0], [(1 << 31) - 1, -(1 << 31), 11, -1], [3, 3, 3, 3]], np.int32)
    w = np.where((places >= 0) & (places < 12), 0.5, np.nan).astype(np.float32)
    ob, pb, wb, y = hip.put(o), hip.put(places), hip.put(w), hip.full((T, H), 7.0)
    d = moe.Dispatch(9, K, H, moe.QT_F32)
    d.combine_async(ob.ptr, T, pb.ptr, y.ptr, wb.ptr)
    assert np.allclose(y.get(), [o[0], o[11] / 2, 2 * o[3]], rtol=2.0 ** -22)
    dw, dout = hip.full((T, K), 7.0), hip.full((T * K, H), 7.0)
    d.combine_backward_async(ob.ptr, T, pb.ptr, ob.ptr, dout.ptr, dw.ptr, wb.ptr)
    got = dw.get()
    assert (got[[0, 0, 1, 1, 1], [1, 2, 0, 1, 3]] == 0).all()
    there = np.zeros(T * K, bool)
    there[[0, 11, 3]] = True
    assert (dout.get()[~there] == 7.0).all() and np.allclose(dout.get()[11], o[1] / 2)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,K,E,H", BACK)
def test_combine_backward(T, K, E, H, type):
    for extra, weighted in ((0, True), (3, False)):
        say("combine backward", T, K, E, H, type, extra, weighted)
        places, o, w, pb, ob, wb = back(T, K, E, H, type, extra, T + H + 1, weighted)
        dyb, dy = hip.rows(np.random.default_rng(T).normal(size=(T, H)), type, extra)
        dout, _ = hip.rows(np.full((T * K, H), 7.0), type, extra, 1, 7.0)
        dw = hip.full(T * K + 1, 7.0)
        d = moe.Dispatch(E, K, H, TYPES[type])
        s = H + extra

        def call(dout, dw):
            d.combine_backward_async(dyb.ptr, T, pb.ptr, ob.ptr, dout and dout.ptr, dw and dw.ptr, wb and wb.ptr, dy_stride=s,
                                     o_stride=s, dout_stride=s)

        call(dout, dw)
        got, gw = decode(dout.get(), type), dw.get()
        assert gw[-1] == 7.0
        t, k = np.nonzero(places >= 0)
        p = places[t, k]
        want = dy[t] * (w[t, k].astype(np.float64)[:, None] if weighted else 1.0)
        assert (np.abs(got[p, :H] - want) <= (ref.EPS[type] + 2.0 ** -24) * 1.0001 * np.abs(want) + TINY[type]).all()
        rest = np.setdiff1d(np.arange(len(got)), p)
        assert (got[rest] == 7.0).all() and (got[:, H:] == 7.0).all()
        want = np.zeros((T, K))
        want[t, k] = (dy[t] * o[p]).sum(-1)
        size = np.zeros((T, K))
        size[t, k] = np.abs(dy[t] * o[p]).sum(-1)
        assert (np.abs(gw[:-1].reshape(T, K) - want) <= (H / 64 + 16) * 2.0 ** -24 * size + 2.0 ** -149).all()
        # Each gradient alone: the same bits.
        only, _ = hip.rows(np.full((T * K, H), 7.0), type, extra, 1, 7.0)
        call(only, None)
        assert np.array_equal(only.get(), dout.get())
        alone = hip.full(T * K + 1, 7.0)
        call(None, alone)
        assert np.array_equal(alone.get(), gw)


def test_gradients_by_differences():
    """The calls' gradients of L = sum(c * y), y = combine(o = g * dispatch(x), w), against L's differences in 64 bits."""
    T, K, E, H = 6, 3, 4, 20
    say("differences")
    r = np.random.default_rng(2)
    ids = draw_ids(T, K, E, 9, 0.2)
    order, places, offsets = ref.dispatch(ids, E)
    P = offsets[-1]
    x, w, c = (r.normal(size=s).astype(np.float32).astype(np.float64) for s in ((T, H), (T, K), (T, H)))
    g = r.normal(size=(T * K, H)).astype(np.float32).astype(np.float64)

    def loss(x, w):
        o = np.zeros((T * K, H))
        o[:P] = g[:P] * x[order[:P] // K]
        return (c * ref.combine(o, places, w)[0]).sum(), o

    _, o = loss(x, w)
    d = moe.Dispatch(E, K, H, moe.QT_F32)
    bufs = [hip.put(a.astype(np.float32)) for a in (c, o, w)]
    pb, dout, dw, dx = hip.put(places.astype(np.int32)), hip.full((T * K, H), 0), hip.full((T, K), 0), hip.full((T, H), 0)
    d.combine_backward_async(bufs[0].ptr, T, pb.ptr, bufs[1].ptr, dout.ptr, dw.ptr, bufs[2].ptr)
    dxs = hip.put((dout.get() * g).astype(np.float32))  # the gradient of the experts in between
    d.dispatch_backward_async(dxs.ptr, T, pb.ptr, dx.ptr)
    h = 2.0 ** -10
    for got, v, at in ((dx.get(), x, 0), (dw.get(), w, 1)):
        for i in np.ndindex(v.shape):
            e = np.zeros_like(v)
            e[i] = h
            a = [x, w]
            a[at] = v + e
            up = loss(*a)[0]
            a[at] = v - e
            want = (up - loss(*a)[0]) / (2 * h)  # (L is linear in each: the difference is exact to 2^-40)
            assert abs(got[i] - want) <= 2.0 ** -20 * (1 + H)


def test_graph_streams_and_others_work():
    """There and back with the routing before it, captured and replayed on new tokens between eager calls; two graphs that share
    the buffers replay one after the other."""
    T, K, E, H = 90, 4, 32, 260
    say("graph")
    r = np.random.default_rng(4)
    logits = hip.full((T, E), 0)
    x = hip.full((T, H), 0, np.uint16)
    d, router = moe.Dispatch(E, K, H), moe.Router(E, K)

    def buffers():
        return dict(ids=hip.full((T, K), 0, np.int32), w=hip.full((T, K), 0), xs=hip.full((T * K, H), 0, np.uint16),
                    order=hip.full(T * K, 0, np.int32), places=hip.full((T, K), 0, np.int32), offsets=hip.full(E + 1, 0, np.int32),
                    y=hip.full((T, H), 0, np.uint16), dout=hip.full((T * K, H), 0, np.uint16), dw=hip.full((T, K), 0),
                    dx=hip.full((T, H), 0, np.uint16))

    def forward(b, s):
        router.route_async(logits.ptr, T, b["ids"].ptr, b["w"].ptr, stream=s)
        d.dispatch_async(x.ptr, T, b["ids"].ptr, b["xs"].ptr, b["order"].ptr, b["places"].ptr, b["offsets"].ptr, stream=s)
        d.combine_async(b["xs"].ptr, T, b["places"].ptr, b["y"].ptr, b["w"].ptr, stream=s)

    def backward(b, s):
        d.combine_backward_async(x.ptr, T, b["places"].ptr, b["xs"].ptr, b["dout"].ptr, b["dw"].ptr, b["w"].ptr, stream=s)
        d.dispatch_backward_async(b["dout"].ptr, T, b["places"].ptr, b["dx"].ptr, stream=s)

    a, b = buffers(), buffers()
    s1, s2 = hip.stream(), hip.stream()
    first = hip.capture(s1, lambda: forward(a, s1))
    second = hip.capture(s1, lambda: backward(a, s1))
    for i in range(4):
        logits.put(r.normal(size=(T, E)).astype(np.float32))
        x.put(encode(r.normal(size=(T, H)), "bf16"))
        first()
        second()
        forward(b, s2)
        backward(b, s2)
        for name in a:
            assert np.array_equal(a[name].get(), b[name].get()), name
        order, places, offsets = ref.dispatch(b["ids"].get(), E)
        assert np.array_equal(a["order"].get(), order) and np.array_equal(a["offsets"].get(), offsets)
        v = decode(x.get(), "bf16")
        w = b["w"].get().astype(np.float64)
        want = v * w.sum(-1)[:, None]  # every rank's row is the token's own
        assert (np.abs(decode(a["y"].get(), "bf16") - want) <= (ref.EPS["bf16"] + 2.0 ** -20) * np.abs(want) + 2.0 ** -120).all()


def test_threads():
    """Calls from four threads at once, each on a stream and buffers of its own."""
    say("threads")
    jobs = []
    for i, T in enumerate((2, 60, 1500, 700)):
        ids = draw_ids(T, 8, 64, i, 0.1)
        jobs.append((Call(ids, 64, 96, "bf16", seed=i), ids, hip.stream()))
    threads = [threading.Thread(target=lambda c=c, s=s: [c.run(s) for _ in range(20)]) for c, _, s in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for c, ids, _ in jobs:
        c.check(ids)


def test_no_tokens():
    say("no tokens")
    b = hip.full(9, 7, np.int32)
    d = moe.Dispatch(8, 4, 64)
    d.dispatch_async(None, 0, None, None, None, None, b.ptr)
    assert not b.get().any()


def test_a_device_that_is_not_there():
    """Refused with the runtime's error, which the next call does not see."""
    say("device")
    b = hip.full(64, 0)
    with pytest.raises(moe.MoeError) as e:
        moe.Dispatch(8, 1, 4, device=99).combine_async(b.ptr, 1, b.ptr, b.ptr + 128)
    assert e.value.status == MOE_ERROR
    moe.Dispatch(8, 1, 4).combine_async(b.ptr, 1, b.ptr, b.ptr + 128)
