"""The experts of routed tokens in 8-bit integers, against the plain form in 64 bits within the bound that tests/more_ref.py derives
(and one rounding to the result's type), alone and behind the routing."""
import threading

import numpy as np
import pytest

from tests import more_ref as ref
from tests import ops_ref
from tests.harness import moe
from tests.ops_dev import TYPES, Raw, decode, encode, hip
from tests.test_gpu_i8 import TINY, matrix, room, say

pytestmark = pytest.mark.gpu


class Model:
    def __init__(self, E, H, F, seed, sigma=0.05):
        r = np.random.default_rng(seed)
        self.E, self.H, self.F, self.hold = E, H, F, []
        self.m, self.v = [], []
        for rows, cols in ((F, H), (F, H), (H, F)):
            codes, scales = ref.i8_quantize((r.normal(size=(E * rows, cols)) * sigma).astype(np.float32))
            m, c, s = matrix(E * rows, cols, codes, scales)
            self.hold += [(ref.i8_padded(codes), c), (scales.astype(np.float32), s)]
            self.m.append(moe.I8Matrix(m.codes, m.scales, rows, cols))
            self.v.append((codes.reshape(E, rows, cols), scales.reshape(E, rows)))

    def op(self, K, x="f32", y="f32", limit=0.0):
        return moe.I8Experts(self.H, self.F, self.E, K, *self.m, x_type=TYPES[x], y_type=TYPES[y], swiglu_limit=limit)


def run(model, x, ids, w, type="f32", out="f32", limit=0.0, extra=0):
    T, K = ids.shape
    H = model.H
    xb, values = hip.rows(x, type, extra)
    idb, wb = hip.put(ids.astype(np.int32)), hip.put(w.astype(np.float32))
    y, _ = hip.rows(np.full((T, H), 7.0), out, extra, 1, 7.0)
    op = model.op(K, type, out, limit)
    n = op.work_bytes(T)
    work = room(n + 64)
    op.forward_async(xb.ptr, T, idb.ptr, wb.ptr, y.ptr, work.ptr, n, x_stride=H + extra, y_stride=H + extra)
    got = decode(y.get(), out)
    assert (got[T:] == 7.0).all() and (got[:, H:] == 7.0).all() and (work.get()[n:] == 0xA5).all()
    return got[:T, :H], values


def within(got, y, off, out="f32"):
    off = off + ref.EPS[out] * (np.abs(y) + off) + TINY[out]
    assert np.all(np.abs(got - y) <= off), float((np.abs(got - y) / off).max())


def check(model, x, ids, w, type="f32", out="f32", limit=0.0, extra=0, rows=slice(None)):
    got, values = run(model, x, ids, w, type, out, limit, extra)
    w = w.astype(np.float32).astype(np.float64)
    within(got[rows], *ref.i8_experts(values[rows], ids[rows], w[rows], *model.v, limit=limit), out)
    return got


def tokens(T, H, E, K, seed, dropped=0.0, repeat=False):
    r = np.random.default_rng(seed)
    x = r.normal(size=(T, H)).astype(np.float32)
    ids = r.integers(0, E, size=(T, K)) if repeat else np.array([r.permutation(E)[:K] for _ in range(T)]).reshape(T, K)
    ids = np.where(r.random((T, K)) < dropped, -1, ids)
    return x, ids, r.random((T, K))


@pytest.mark.parametrize("T,H,F,E,K", [(1, 128, 32, 4, 2), (1, 1000, 200, 8, 3), (1, 512, 256, 16, 10), (2, 33, 7, 3, 1),
                                       (5, 640, 96, 32, 6), (8, 256, 160, 64, 8), (16, 512, 128, 8, 4), (17, 256, 96, 16, 4),
                                       (33, 1, 1, 2, 2), (40, 384, 128, 4, 4), (70, 320, 260, 5, 2), (150, 256, 64, 3, 2),
                                       (9, 2560, 640, 6, 4), (300, 130, 129, 40, 5),
                                       (16, 256, 600, 12, 10), (23, 256, 64, 12, 7), (16, 200, 700, 12, 10),
                                       (3, 2100, 64, 4, 2), (20, 3200, 96, 2, 2), (200, 640, 640, 64, 2), (90, 384, 300, 4, 2),
                                       (2, 2700, 129, 3, 3), (13, 5200, 24, 2, 2), (1, 300, 5000, 3, 2), (16, 256, 500, 200, 10),
                                       (16, 2100, 500, 40, 10), (12, 300, 640, 8, 8), (11, 128, 899, 100, 7)])
def test_experts(T, H, F, E, K):
    say("experts", T, H, F, E, K)
    model = Model(E, H, F, T + H)
    check(model, *tokens(T, H, E, K, T))
    check(model, *tokens(T, H, E, K, T + 1, 0.3, True), limit=0.05, extra=3)


@pytest.mark.parametrize("T,H,F,E,K,skew", [(1100, 64, 40, 100, 4, 0.0), (1100, 64, 40, 100, 4, 0.9), (1050, 5700, 40, 8, 4, 0.0),
                                            (600, 2300, 8, 512, 4, 0.0), (600, 2300, 8, 300, 8, 0.0)])
def test_many(T, H, F, E, K, skew):
    """Several slices of ids, several blocks of columns an item, most tokens on one expert."""
    say("many", T, H, F, E, K, skew)
    x, ids, w = tokens(T, H, E, K, 7, 0.05)
    ids[np.random.default_rng(1).random(T) < skew, 0] = E - 1
    check(Model(E, H, F, 5), x, ids, w, rows=np.r_[0:20, T // 2:T // 2 + 20, T - 20:T])


@pytest.mark.parametrize("T,H,F,E,K,limit", [(600, 600, 640, 100, 4, 0.0), (600, 520, 640, 100, 4, 0.1), (2500, 260, 640, 100, 4, 0.0),
                                             (2500, 100, 640, 100, 4, 0.1), (2500, 1300, 130, 100, 4, 0.0), (250, 1030, 260, 250, 2, 0.0)])
def test_several_items_a_work_group(T, H, F, E, K, limit):
    """More pieces of tiles than work-groups, with 32, 64 and 128 rows, of one stage to eleven."""
    say("items", T, H, F, E, K, limit)
    check(Model(E, H, F, 4), *tokens(T, H, E, K, 8, 0.05), limit=limit, rows=np.r_[0:16, T // 2:T // 2 + 16, T - 16:T])


@pytest.mark.parametrize("T", [2, 40])
def test_large_gates(T):
    """Gates of hundreds to both sides: the SiLU at its ends."""
    say("large gates", T)
    check(Model(6, 512, 96, 8, sigma=5.0), *tokens(T, 512, 6, 3, 5))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T", [1, 6, 50])
def test_types(T, type, out):
    say("types", T, type, out)
    check(Model(8, 512, 160, 3), *tokens(T, 512, 8, 3, T, 0.1), type=type, out=out, extra=8)


@pytest.mark.parametrize("T", [1, 7, 64, 200])
def test_ids(T):
    """Every token on one expert; none at all; ids out of range; the same expert in each rank."""
    say("ids", T)
    model = Model(6, 256, 96, 8)
    x, ids, w = tokens(T, 256, 6, 4, 5)
    check(model, x, np.full((T, 1), 5), w[:, :1])
    got = check(model, x, np.full((T, 4), -1), w)
    assert not got.any()
    far = ids.copy()
    far[:, 0], far[:, 1], far[::2, 2] = 6, -(1 << 31), (1 << 31) - 1
    check(model, x, far, w)
    check(model, x, np.repeat(ids[:, :1], 4, 1), w)
    check(model, x, ids, np.where(w < 0.5, 0.0, -w))


@pytest.mark.parametrize("T", [3, 12, 100, 900])
def test_padded_batch_and_nans(T):
    """Tokens that stand for nothing (no expert, rows and weights of NaNs) get zeros and change nobody else's result; a token with
    a NaN or an infinity gets NaNs and changes nobody else's."""
    say("padded", T)
    model = Model(6, 256, 96, 8)
    x, ids, w = tokens(T, 256, 6, 2, 5)
    clean, _ = run(model, x, ids, w)
    pad = np.arange(T) % 3 == 1
    x[pad], ids[pad], w[pad] = np.nan, -1, np.nan
    x[0, 200], x[2, 3] = np.nan, np.inf
    got, _ = run(model, x, ids, w)
    bad = np.arange(T) % T < 3
    bad[1] = False
    assert not got[pad].any() and np.isnan(got[bad]).all()
    assert np.array_equal(got[~pad & ~bad], clean[~pad & ~bad])


def chain(model, x, T, wr, K, work, out, stream):
    """Logits by the dense product, the routing, the experts: as a layer calls them."""
    E = model.E
    logits, ids, w, load, y = out
    moe.i8_linear_async(moe.QT_BF16, x.ptr, T, wr, moe.QT_F32, logits.ptr, work[0].ptr, work[0].nbytes, stream=stream)
    moe.Router(E, K, moe.MOE_SCORE_SIGMOID, 4, 2, 2).route_async(logits.ptr, T, ids.ptr, w.ptr, load.ptr, stream=stream)
    model.op(K, "bf16", "bf16").forward_async(x.ptr, T, ids.ptr, w.ptr, y.ptr, work[1].ptr, work[1].nbytes, stream=stream)


@pytest.mark.parametrize("T", [1, 8, 90])
def test_chain_and_graph(T):
    """The operators together, eager against the plain forms, then captured and replayed on new tokens between eager calls."""
    say("chain", T)
    E, H, F, K = 16, 512, 96, 4
    model = Model(E, H, F, 21)
    r = np.random.default_rng(T)
    wf = hip.put((r.normal(size=(E, H)) * 0.1).astype(np.float32))
    wr, c, s = matrix(E, H)
    moe.i8_quantize_async(moe.QT_F32, wf.ptr, wr)
    x = hip.full((T, H), 0, np.uint16)
    work = [[room(moe.i8_linear_work_bytes(wr, T) + 16), room(model.op(K).work_bytes(T))] for _ in range(2)]

    def outputs():
        return [hip.full((T, E), 0), hip.full((T, K), 0, np.int32), hip.full((T, K), 0), hip.full(E, 0, np.int32),
                hip.full((T, H), 0, np.uint16)]

    a, b = outputs(), outputs()
    s1, s2 = hip.stream(), hip.stream()
    x.get()  # (the quantisation is done)
    launch = hip.capture(s1, lambda: chain(model, x, T, wr, K, work[0], a, s1))
    for i in range(4):
        x.put(encode(r.normal(size=(T, H)), "bf16"))
        launch()
        chain(model, x, T, wr, K, work[1], b, s2)
        for u, v in zip(a, b):
            assert np.array_equal(u.get(), v.get())
        ids, w, load = ops_ref.route(b[0].get(), K, True, None, 4, 2, 2)
        assert np.array_equal(b[1].get(), ids) and np.array_equal(b[3].get(), load)
        y, off = ref.i8_experts(decode(x.get(), "bf16"), ids, b[2].get().astype(np.float64), *model.v)
        within(decode(b[4].get(), "bf16"), y, off, "bf16")


def test_dispatched_rows_give_the_experts_result():
    """The experts' steps by the other operators: rows dispatched, each expert's products on its own rows, combined. The same
    quantisations, sums and order of ranks: y within the SiLU's roundings, which the bound holds."""
    say("by steps")
    T, E, H, F, K = 60, 8, 256, 96, 3
    model = Model(E, H, F, 2)
    x, ids, w = tokens(T, H, E, K, 1, 0.1)
    d = moe.Dispatch(E, K, H, moe.QT_F32)
    n = T * K
    xb, idb, wb = hip.put(x), hip.put(ids.astype(np.int32)), hip.put(w.astype(np.float32))
    xs, o, y = hip.full((n, H), 0), hip.full((n, H), np.nan), hip.full((T, H), 7.0)
    order, places, offsets = hip.full(n, 0, np.int32), hip.full(n, 0, np.int32), hip.full(E + 1, 0, np.int32)
    d.dispatch_async(xb.ptr, T, idb.ptr, xs.ptr, order.ptr, places.ptr, offsets.ptr)
    at = offsets.get()
    work = room(1 << 20)
    for e in range(E):
        a, m = int(at[e]), int(at[e + 1] - at[e])
        g, u = hip.full((m, F), 0), hip.full((m, F), 0)
        gate, up, down = (moe.I8Matrix(mm.codes + e * mm.rows * ref.pad128(mm.cols), mm.scales + 4 * e * mm.rows, mm.rows, mm.cols)
                          for mm in model.m)
        for wm, to in ((gate, g), (up, u)):
            moe.i8_linear_async(moe.QT_F32, xs.ptr + a * H * 4, m, wm, moe.QT_F32, to.ptr, work.ptr, work.nbytes)
        gv = g.get().astype(np.float64)
        h = hip.put((gv / (1 + np.exp(-gv)) * u.get()).astype(np.float32))
        moe.i8_linear_async(moe.QT_F32, h.ptr, m, down, moe.QT_F32, o.ptr + a * H * 4, work.ptr, work.nbytes)
        o.get()  # (h lives until the product is done)
    d.combine_async(o.ptr, T, places.ptr, y.ptr, wb.ptr)
    want, off = ref.i8_experts(x, ids, w.astype(np.float32).astype(np.float64), *model.v)
    within(y.get(), want, off)
    within(run(model, x, ids, w)[0], want, off)


def test_threads_and_streams():
    """Calls from four threads at once, each on a stream and buffers of its own, few and many tokens."""
    say("threads")
    model = Model(12, 256, 96, 4)
    jobs = []
    for i, T in enumerate((1, 30, 200, 9)):
        x, ids, w = tokens(T, 256, 12, 4, i, 0.1)
        want = run(model, x, ids, w)[0]
        op, s = model.op(4), hip.stream()
        bufs = [hip.put(x), hip.put(ids.astype(np.int32)), hip.put(w.astype(np.float32)), hip.full((T, 256), 7.0),
                room(op.work_bytes(T))]
        jobs.append((op, T, s, bufs, want))

    def call(op, T, s, b):
        for _ in range(20):
            op.forward_async(b[0].ptr, T, b[1].ptr, b[2].ptr, b[3].ptr, b[4].ptr, b[4].nbytes, stream=s)

    threads = [threading.Thread(target=call, args=j[:4]) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for op, T, s, b, want in jobs:
        assert np.array_equal(b[3].get(), want)


def test_far_experts():
    """Matrices past 2^32 bytes: the last expert's."""
    say("far experts")
    E, H, F = 512, 16384, 640  # 512 x 640 x 16384 bytes: 5.4 GB a matrix
    model = Model(1, H, F, 2)
    far = Model.__new__(Model)
    far.E, far.H, far.F, far.m, far.hold = E, H, F, [], []
    for i, (rows, cols) in enumerate(((F, H), (F, H), (H, F))):
        parts = []
        for host, _ in model.hold[2 * i:2 * i + 2]:
            b = Raw(hip, E * host.nbytes)
            b.put(host.ravel().view(np.uint8), (E - 1) * host.nbytes)
            parts.append(b)
        far.hold += parts
        far.m.append(moe.I8Matrix(parts[0].ptr, parts[1].ptr, rows, cols))
    for T in (1, 20, 200):
        x, _, w = tokens(T, H, 2, 1, 3)
        got, values = run(far, x, np.full((T, 1), E - 1), w)
        rows = np.arange(T)[-20:]
        within(got[rows], *ref.i8_experts(values[rows], np.zeros((len(rows), 1), int), w[rows].astype(np.float32).astype(np.float64), *model.v))


def test_far_positions():
    """The most tokens and ranks: rows of h past 2^32 bytes, their codes past 2^30."""
    say("far positions")
    T, H, F, E, K = 16384, 64, 5000, 20, 16
    check(Model(E, H, F, 6), *tokens(T, H, E, K, 9, 0.01), rows=np.r_[0:8, T // 2:T // 2 + 8, T - 24:T])


@pytest.mark.parametrize("T,H,F,E,K", [(4096, 2300, 40, 20, 16), (4200, 2300, 8, 400, 8)])
def test_columns_in_parts(T, H, F, E, K):
    """More values than down takes at a time: three parts of 768 columns (2304 of 65536 assignments are 604 MB), and parts of 1280
    and 1024; n_embd ends inside the last."""
    say("columns in parts", T, H, F, E, K)
    check(Model(E, H, F, 6), *tokens(T, H, E, K, 9, 0.05), rows=np.r_[0:16, T // 2:T // 2 + 16, T - 16:T])


@pytest.mark.parametrize("T", [8, 90])
def test_graphs_that_share_a_work_buffer(T):
    """Two captured calls on one work buffer, replayed in turn on one stream, with eager calls and waits between."""
    say("shared work", T)
    model, K = Model(12, 512, 128, 4), 4
    op, s = model.op(K), hip.stream()
    n = op.work_bytes(T)
    work, other = room(n), room(n)
    sets = []
    for seed in (6, 7):
        x, ids, w = tokens(T, 512, 12, K, seed, 0.2)
        b = [hip.put(x), hip.put(ids.astype(np.int32)), hip.put(w.astype(np.float32)), hip.full((T, 512), 7.0)]

        def call(y, room, stream, b=b):
            op.forward_async(b[0].ptr, T, b[1].ptr, b[2].ptr, y.ptr, room.ptr, n, stream=stream)

        sets.append((b, call, hip.capture(s, lambda call=call, b=b: call(b[3], work, s))))
    r, eager = np.random.default_rng(3), hip.full((T, 512), 0)
    for _ in range(3):
        for b, _, _ in sets:
            b[0].put(r.normal(size=(T, 512)).astype(np.float32))
        for _, _, launch in sets:
            launch()
        for b, call, _ in sets:
            call(eager, other, None)
            assert np.array_equal(b[3].get(), eager.get())


def test_no_tokens():
    say("no tokens")
    model = Model(4, 128, 32, 1)
    y = hip.full((2, 128), 7)
    model.op(2).forward_async(y.ptr, 0, y.ptr, y.ptr, y.ptr, None, 0)
    assert (y.get() == 7.0).all()


@pytest.mark.parametrize("T", [1, 12, 100, 900])
def test_whatever_the_work_buffer_held(T):
    """Zeros, bytes whose floats, codes and counts are NaNs and -1, and what another batch left: the same bits. Ranks without an
    expert leave rows of the work unwritten."""
    say("work buffer", T)
    model, K = Model(12, 512, 128, 4), 4
    op = model.op(K)
    n = op.work_bytes(T)
    work = room(n)
    batches = []
    for seed in (6, 7):
        x, ids, w = tokens(T, 512, 12, K, seed, 0.3)
        batches.append((hip.put(x), hip.put(ids.astype(np.int32)), hip.put(w.astype(np.float32)), hip.full((T, 512), 7.0)))

    def call(b):
        x, ids, w, y = batches[b]
        op.forward_async(x.ptr, T, ids.ptr, w.ptr, y.ptr, work.ptr, n)
        return y.get()

    got = []
    for value in (0x00, 0xFF, 0x7F):
        work.put(np.full(n, value, np.uint8))
        got.append(call(0))
    call(1)
    got.append(call(0))
    assert np.isfinite(got[0]).all()
    assert all(np.array_equal(got[0], g) for g in got[1:])


@pytest.mark.parametrize("T", [2, 12, 100, 900])
def test_a_token_whatever_the_others(T):
    """Batches of one size that share some tokens: these have the same bits, whoever uses their experts beside them."""
    say("a token's own", T)
    model = Model(12, 512, 128, 4)
    (x, ids, w), (x2, ids2, w2) = (tokens(T, 512, 12, 4, s, 0.2) for s in (6, 7))
    ids2[:] = np.where(np.arange(T)[:, None] % 2, ids2, 3)  # half of them on one expert
    same = np.r_[T // 2, T - 1]
    x2[same], ids2[same], w2[same] = x[same], ids[same], w[same]
    assert np.array_equal(run(model, x, ids, w)[0][same], run(model, x2, ids2, w2)[0][same])
